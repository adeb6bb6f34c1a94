"""Paged serving operators on the GPU against plain 64-bit forms.

Tolerances come from the arithmetic: u = 2^-24 is half an f32 ulp, half = half an ulp of the output type.
- rope: the mean of squares adds D terms (relative error D u at most, halved by the root), a few more
  roundings follow, and the output is rounded once: half |y| + (D / 2 + 8) u max|row|.
- attention: a score's error is at most (D + 2) u scale sum|q k|; it enters twice (through a weight and
  through the sum of weights); sums of n terms add (n + 16) u; queries of 16 bits round the weights of the
  second product to their type (half of its ulp); all of it times max|v|, and the output is rounded once.
- sampling: the drawn id must lie where the 64-bit running share holds u to within 2^-20 (weights are good
  to about 2^-22 of themselves), the kept set is exact wherever no 64-bit share is that near to top_p.
"""
import math

import numpy as np
import pytest

from conftest import pkg

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of an output's ulp, relative (bf16: 8 bits of significand)


def _torch(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Pool:
    """A page pool of random values, NaN in every page that no sequence owns and past every length."""

    def __init__(self, lens, page, hk, dim, cache, layout="head", spare=3, seed=0, gap=0, width=0):
        import torch
        rng = np.random.default_rng(seed)
        self.lens, self.page, self.hk, self.dim, self.cache, self.layout = list(lens), page, hk, dim, cache, layout
        need = [-(-n // page) for n in lens]
        self.n = sum(need) + spare
        order = rng.permutation(self.n).astype(np.int32)
        self.table = np.full((len(lens), max([width, 1] + need)), -7, np.int32)
        at = 0
        for i, m in enumerate(need):
            self.table[i, :m] = order[at: at + m]
            at += m
        shape = (self.n, hk, page) if layout == "head" else (self.n, page, hk)
        t = _torch(cache)
        self.full = [torch.full(shape + (dim + gap,), math.nan, dtype=t, device="cuda") for _ in range(2)]
        for i, n in enumerate(lens):
            for p0 in range(0, n, page):
                m = min(page, n - p0)
                for f in self.full:
                    x = torch.from_numpy(rng.standard_normal((hk, m, dim)).astype(np.float32)).cuda().to(t)
                    pg = self.table[i, p0 // page]
                    if layout == "head":
                        f[pg, :, :m, :dim] = x
                    else:
                        f[pg, :m, :, :dim] = x.transpose(0, 1)
        st = self.full[0].stride()
        self.kv = pkg().paged_kv(self.full[0].data_ptr(), self.full[1].data_ptr(), cache, self.n, page, hk, dim,
                                 (st[0], st[1], st[2]) if layout == "head" else (st[0], st[2], st[1]))
        self.d_table = torch.from_numpy(self.table).cuda()
        self.d_len = torch.from_numpy(np.array(lens, np.int32)).cuda()

    def rows(self, which, seq, n):
        """[kv head][n][dim] of sequence seq in 64 bits."""
        f = self.full[which].double().cpu().numpy()[..., : self.dim]
        if self.layout == "pos":
            f = f.transpose(0, 2, 1, 3)
        if n == 0:
            return np.zeros((self.hk, 0, self.dim))
        return np.concatenate([f[pg] for pg in self.table[seq, : -(-n // self.page)]], 1)[:, :n]


def _attend(pool, act, heads, scale, seed=1, lse=True, stream=0, d_len=None, q_gap=0, q=None):
    import torch
    P = pkg()
    b, dim = len(pool.lens), pool.dim
    if q is None:
        q = np.random.default_rng(seed).standard_normal((b, heads, dim)).astype(np.float32)
    wide = torch.zeros(b, heads * dim + q_gap, device="cuda", dtype=_torch(act))
    wide[:, : heads * dim] = torch.from_numpy(q.reshape(b, -1)).cuda().to(_torch(act))
    out = torch.full((b, heads * dim + q_gap), 7.0, device="cuda", dtype=_torch(act))
    ls = torch.full((b, heads), 7.0, device="cuda") if lse else None
    ws = torch.zeros(P.paged_attn_workspace(b, heads, dim), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    res = []
    for _ in range(2):  # the second call finds the workspace as the first left it
        P.paged_attn_device(pool.kv, act, wide.data_ptr(), wide.stride(0), b, heads, (pool.d_len if d_len is None else d_len).data_ptr(),
                            pool.d_table.data_ptr(), pool.d_table.stride(0), scale, out.data_ptr(), out.stride(0), ws.data_ptr(),
                            ws.numel(), ls.data_ptr() if lse else 0, stream)
        torch.cuda.synchronize()
        res.append((out.clone(), ls.clone() if lse else None))
    assert torch.equal(res[0][0].view(torch.uint8), res[1][0].view(torch.uint8))  # same bits again
    if q_gap:
        assert (out[:, heads * dim:] == 7.0).all()
    return (wide[:, : heads * dim].double().cpu().numpy().reshape(b, heads, dim),
            out[:, : heads * dim].double().cpu().numpy().reshape(b, heads, dim), ls.double().cpu().numpy() if lse else None)


def _check_attention(pool, act, heads, scale, **kw):
    q, out, lse = _attend(pool, act, heads, scale, **kw)
    for s, n in enumerate(pool.lens):
        k, v = pool.rows(0, s, n), pool.rows(1, s, n)
        if n == 0:
            assert (out[s] == 0).all() and (lse is None or (lse[s] == -np.inf).all())
            continue
        for h in range(heads):
            hk = h // (heads // pool.hk)
            x = scale * (k[hk] @ q[s, h])
            m = x.max()
            e = np.exp(x - m)
            ref, ref_l = e @ v[hk] / e.sum(), m + math.log(e.sum())
            ds = (pool.dim + 2) * U * (abs(scale) * np.abs(k[hk]) @ np.abs(q[s, h])).max()
            weights = 0.0 if act == "f32" else HALF[act]
            tol = (2 * ds + (n + 16) * U + weights) * np.abs(v[hk]).max()
            assert (np.abs(out[s, h] - ref) <= tol + HALF[act] * np.abs(ref)).all(), (s, h, n, np.abs(out[s, h] - ref).max(), tol)
            if lse is not None:
                assert abs(lse[s, h] - ref_l) <= ds + (n + 16) * U + 4 * U * abs(ref_l), (s, h, n, lse[s, h], ref_l)


KINDS = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f16")]


@pytest.mark.parametrize("act,cache", KINDS)
@pytest.mark.parametrize("dim", [8, 32, 64, 80, 96, 128, 200, 256])
def test_attention_head_sizes(act, cache, dim, cuda_ok):
    pool = Pool([0, 1, 5, 16, 17, 130, 333], 16, 2, dim, cache, seed=dim)
    _check_attention(pool, act, 6, dim ** -0.5)


@pytest.mark.parametrize("act,cache", KINDS)
@pytest.mark.parametrize("hk,rep", [(1, 1), (3, 3), (5, 2), (1, 7), (2, 8), (1, 9), (2, 16), (1, 17), (1, 64)])
def test_attention_head_groups(act, cache, hk, rep, cuda_ok):
    pool = Pool([63, 64, 65, 0, 200], 32, hk, 64, cache, seed=rep)
    _check_attention(pool, act, hk * rep, 0.125)


@pytest.mark.parametrize("act,cache", KINDS)
@pytest.mark.parametrize("page,layout", [(1, "head"), (1, "pos"), (3, "pos"), (7, "head"), (16, "pos"), (24, "head"), (100, "pos"),
                                         (256, "head")])
def test_attention_page_sizes_and_layouts(act, cache, page, layout, cuda_ok):
    pool = Pool([1, 2, 3, 8, 99, 100, 101, 257], page, 3, 64, cache, layout, seed=page, width=300)
    _check_attention(pool, act, 9, 0.125)


@pytest.mark.parametrize("act,cache", KINDS)
def test_attention_gaps_between_rows_and_queries(act, cache, cuda_ok):
    pool = Pool([40, 77], 16, 2, 64, cache, "pos", gap=8, seed=3)
    _check_attention(pool, act, 4, 0.125, q_gap=16)
    _check_attention(pool, act, 4, 0.125, lse=False)


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("lens,hk,dim", [([9001], 1, 64), ([5000, 0, 3, 4097], 2, 128), ([2500] + [1] * 40 + [0] * 20, 1, 64),
                                         ([700] * 33, 3, 64)])
def test_attention_long_and_ragged(act, cache, lens, hk, dim, cuda_ok):
    _check_attention(Pool(lens, 64, hk, dim, cache, seed=9), act, hk * 3, dim ** -0.5)


@pytest.mark.parametrize("seqs,offset", [(31, 0), (33, 1), (130, 3), (300, 2), (1100, 1)])
def test_attention_many_sequences_and_lengths_anywhere(seqs, offset, cuda_ok):
    """More sequences than lanes, and lengths that do not begin on a 16-byte boundary."""
    import torch
    rng = np.random.default_rng(seqs)
    lens = np.where(rng.random(seqs) < 0.1, 0, rng.integers(1, 90, seqs))
    lens[rng.integers(seqs)] = 700
    pool = Pool(lens.tolist(), 16, 1, 64, "bf16", seed=seqs)
    d_len = torch.zeros(seqs + 4, dtype=torch.int32, device="cuda")[offset: offset + seqs]
    d_len.copy_(pool.d_len)
    _check_attention(pool, "bf16", 2, 0.125, d_len=d_len)


def test_attention_scores_far_apart(cuda_ok):
    """Scores to +-1e4: the running maximum jumps in every direction and most weights vanish."""
    for act, cache in KINDS:
        pool = Pool([300, 1000], 16, 1, 64, cache, seed=5)
        _check_attention(pool, act, 3, 100.0)
        _check_attention(pool, act, 3, -100.0)
        _check_attention(pool, act, 3, 0.0)


@pytest.mark.parametrize("act,cache", KINDS)
def test_attention_infinite_scores(act, cache, cuda_ok):
    """A key of -inf leaves its position out; a sequence of only such keys is empty; a NaN in use shows."""
    import torch
    pool = Pool([40, 33, 20], 16, 1, 64, cache, seed=6)
    q = np.abs(np.random.default_rng(0).standard_normal((3, 2, 64))).astype(np.float32) + 0.5
    pg = pool.table
    pool.full[0][pg[0, 1], 0, 3, 0] = -math.inf          # position 19 of sequence 0
    for p in range(33):
        pool.full[0][pg[1, p // 16], 0, p % 16, 5] = -math.inf
    pool.full[0][pg[2, 0], 0, 7, 1] = math.nan
    qd, out, lse = _attend(pool, act, 2, 0.125, q=q)
    k, v = pool.rows(0, 0, 40)[0], pool.rows(1, 0, 40)[0]
    use = np.arange(40) != 19
    for h in range(2):
        x = 0.125 * (k[use] @ qd[0, h])
        e = np.exp(x - x.max())
        ref = e @ v[use] / e.sum()
        ds = 66 * U * (0.125 * np.abs(k[use]) @ np.abs(qd[0, h])).max()
        tol = (2 * ds + 56 * U + (0.0 if act == "f32" else HALF[act])) * np.abs(v).max()
        assert (np.abs(out[0, h] - ref) <= tol + HALF[act] * np.abs(ref)).all()
    assert (out[1] == 0).all() and (lse[1] == -np.inf).all()
    assert np.isnan(out[2]).all() and np.isnan(lse[2]).all()
    assert torch.isfinite(torch.from_numpy(out[:2])).all()


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("bf16", "bf16")])
def test_attention_bad_tables_and_lengths_show(act, cache, cuda_ok):
    """A page id outside the pool, or a length past the table, gives NaN for that sequence alone; a negative
    length is an empty one."""
    import torch
    pool = Pool([40, 40, 40, 40, 40], 16, 1, 64, cache, seed=8)
    pool.d_table[0, 1] = pool.n
    pool.d_table[1, 2] = -1
    d_len = torch.tensor([40, 40, 49, -5, 40], dtype=torch.int32, device="cuda")  # three pages hold 48
    _, out, lse = _attend(pool, act, 2, 0.125, d_len=d_len)
    for s in (0, 1, 2):
        assert np.isnan(out[s]).all() and np.isnan(lse[s]).all()
    assert (out[3] == 0).all() and (lse[3] == -np.inf).all()
    assert np.isfinite(out[4]).all()


def test_attention_offsets_past_32_bits(cuda_ok):
    """Pages whose elements lie more than 2^32 elements into the pool."""
    import torch
    P = pkg()
    big = torch.zeros((1 << 32) + (1 << 21), dtype=torch.float16, device="cuda")
    page_stride = 1 << 20
    n_pages = big.numel() // page_stride
    kv = P.paged_kv(big.data_ptr(), big.data_ptr() + 2 * 16 * 64, "f16", n_pages, 16, 1, 64, (page_stride, 16 * 64, 64))
    x = torch.randn(2, 16, 64, device="cuda").half()
    far = n_pages - 2
    big[far * page_stride: far * page_stride + 2048] = x.reshape(-1)
    table = torch.tensor([[far]], dtype=torch.int32, device="cuda")
    ln = torch.tensor([16], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 64, device="cuda").half()
    out = torch.empty_like(q)
    ws = torch.zeros(P.paged_attn_workspace(1, 1, 64), dtype=torch.uint8, device="cuda")
    P.paged_attn_device(kv, "f16", q.data_ptr(), 64, 1, 1, ln.data_ptr(), table.data_ptr(), 1, 0.125, out.data_ptr(), 64,
                        ws.data_ptr(), ws.numel())
    w = torch.softmax(0.125 * (x[0].double() @ q[0].double()), 0)
    ref = w @ x[1].double()
    tol = (2 * 66 * U * 64 + 32 * U + 2 * HALF["f16"]) * float(x[1].abs().max())
    assert (out[0].double() - ref).abs().max() <= tol


def test_attention_on_a_stream_and_in_a_graph(cuda_ok):
    """The call is captured and replayed with other lengths and contents."""
    import torch
    P = pkg()
    pool = Pool([90, 17, 300], 16, 3, 64, "bf16", seed=11)
    q = torch.randn(3, 9, 64, device="cuda").bfloat16()
    out, lse = torch.empty_like(q), torch.empty(3, 9, device="cuda")
    ws = torch.zeros(P.paged_attn_workspace(3, 9, 64), dtype=torch.uint8, device="cuda")

    def call(stream):
        P.paged_attn_device(pool.kv, "bf16", q.data_ptr(), q.stride(0), 3, 9, pool.d_len.data_ptr(), pool.d_table.data_ptr(),
                            pool.d_table.stride(0), 0.125, out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), lse.data_ptr(), stream)

    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    call(st.cuda_stream)
    st.synchronize()
    first = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        call(torch.cuda.current_stream().cuda_stream)
    for n in ([90, 17, 300], [1, 0, 299]):
        pool.d_len.copy_(torch.tensor(n, dtype=torch.int32))
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        call(0)
        torch.cuda.synchronize()
        assert torch.equal(got, out)
        if n[0] == 90:
            assert torch.equal(got, first)


# ---- rotation into the cache

def _rope_ref(x, gain, eps, cs, sn, rope_dim, interleaved):
    x = x.copy()
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain
    y = x.copy()
    half = rope_dim // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        y[..., a] = x[..., a] * cs[i] - x[..., b] * sn[i]
        y[..., b] = x[..., b] * cs[i] + x[..., a] * sn[i]
    return y


@pytest.mark.parametrize("act,cache", KINDS)
@pytest.mark.parametrize("dim,rope_dim", [(64, 64), (64, 40), (128, 128), (80, 80), (96, 48), (256, 64), (8, 2), (32, 0), (200, 200),
                                          (256, 256), (72, 44)])
@pytest.mark.parametrize("interleaved,norm", [(False, False), (True, True), (False, True), (True, False)])
def test_rope_append(act, cache, dim, rope_dim, interleaved, norm, cuda_ok):
    import torch
    P = pkg()
    heads, hk, page = 6, 2, 16
    for layout, alias in (("head", False), ("pos", True)):
        lens = [1, 40, 16]
        pool = Pool(lens, page, hk, dim, cache, layout, seed=dim + rope_dim)
        before = [f.clone() for f in pool.full]
        rng = np.random.default_rng(dim)
        seq = np.array([1] * 9 + [0] + [-1] + [2] * 5, np.int32)
        pos = np.array(list(range(20, 29)) + [0] + [3] + list(range(11, 16)), np.int32)
        n, width = len(seq), (heads + 2 * hk) * dim
        qkv = torch.from_numpy(rng.standard_normal((n, width + 8)).astype(np.float32) * 3).cuda().to(_torch(act))
        x = qkv[:, :width].double().cpu().numpy().reshape(n, heads + 2 * hk, dim)
        cs, sn = P.rope_tables(64, rope_dim, 1000.0)
        gains = [rng.standard_normal(dim).astype(np.float32) for _ in range(2)]
        dev = [torch.from_numpy(a).cuda() for a in (seq, pos, cs, sn, gains[0], gains[1])]
        q = qkv if alias else torch.full((n, heads * dim), 7.0, device="cuda", dtype=_torch(act))
        P.rope_append_device(pool.kv, act, qkv.data_ptr(), qkv.stride(0), n, heads, dev[0].data_ptr(), dev[1].data_ptr(),
                             pool.d_table.data_ptr(), 3, pool.d_table.stride(0), dev[2].data_ptr(), dev[3].data_ptr(), 64, rope_dim,
                             q.data_ptr(), q.stride(0), interleaved, dev[4].data_ptr() if norm else 0, dev[5].data_ptr() if norm else 0,
                             1e-5)
        torch.cuda.synchronize()
        got = q[:, : heads * dim].double().cpu().numpy().reshape(n, heads, dim)
        want = [f.clone() for f in before]
        for t in range(n):
            if seq[t] < 0:
                assert (got[t] == (x[t, :heads] if alias else 7.0)).all()
                continue
            tab = (cs[pos[t]].astype(np.float64), sn[pos[t]].astype(np.float64), rope_dim, interleaved)
            rq = _rope_ref(x[t, :heads], gains[0].astype(np.float64) if norm else None, 1e-5, *tab)
            rk = _rope_ref(x[t, heads: heads + hk], gains[1].astype(np.float64) if norm else None, 1e-5, *tab)
            pg, at = pool.table[seq[t], pos[t] // page], pos[t] % page
            where = (pg, slice(None), at) if layout == "head" else (pg, at)
            gk = pool.full[0][where].double().cpu().numpy()
            for r, g, half in ((rq, got[t], HALF[act]), (rk, gk, HALF[cache])):
                tol = half * np.abs(r) + (dim / 2 + 8) * U * np.abs(r).max(-1, keepdims=True) + 1e-30
                assert (np.abs(g - r) <= tol).all(), (t, np.abs(g - r).max())
            # v is only rounded to the cache's type
            want[1][where] = qkv[t, :width].reshape(-1, dim)[heads + hk:].to(_torch(cache))
            want[0][where] = pool.full[0][where]
        for w, f in zip(want, pool.full):  # no other row was touched
            assert torch.equal(torch.nan_to_num(w, nan=9.0), torch.nan_to_num(f, nan=9.0))


def test_rope_append_bad_rows_write_nothing(cuda_ok):
    import torch
    P = pkg()
    pool = Pool([20, 20], 16, 1, 64, "f32", seed=2)
    pool.d_table[1, 1] = pool.n
    seq = torch.tensor([0, 0, 2, 1, 0, 0], dtype=torch.int32, device="cuda")
    pos = torch.tensor([-1, 32, 0, 17, 25, 3], dtype=torch.int32, device="cuda")  # 32: past the table; 25: past n_pos; 3: good
    cs, sn = (torch.from_numpy(a).cuda() for a in P.rope_tables(25, 64))
    qkv = torch.randn(6, 4 * 64, device="cuda")
    q = torch.zeros(6, 128, device="cuda")
    before = [f.clone() for f in pool.full]
    P.rope_append_device(pool.kv, "f32", qkv.data_ptr(), 256, 6, 2, seq.data_ptr(), pos.data_ptr(), pool.d_table.data_ptr(), 2,
                         pool.d_table.stride(0), cs.data_ptr(), sn.data_ptr(), 25, 64, q.data_ptr(), 128)
    torch.cuda.synchronize()
    assert torch.isnan(q[:5]).all() and torch.isfinite(q[5]).all()
    for b, f in zip(before, pool.full):
        b[pool.table[0, 0], :, 3] = f[pool.table[0, 0], :, 3]
        assert torch.equal(torch.nan_to_num(b, nan=9.0), torch.nan_to_num(f, nan=9.0))


# ---- page copies

@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layers,pages,hk,page,dim,n", [(1, 4, 1, 1, 8, 1), (3, 64, 2, 16, 64, 20), (2, 5000, 1, 3, 8, 2300),
                                                        (5, 9, 3, 7, 72, 4), (30, 40, 3, 16, 64, 2), (1, 6, 8, 128, 128, 3)])
def test_copy_pages(cache, layers, pages, hk, page, dim, n, cuda_ok):
    import torch
    P = pkg()
    pools = [torch.randn(layers, pages, hk, page, dim, device="cuda").to(_torch(cache)) for _ in range(2)]
    want = [p.clone() for p in pools]
    order = np.random.default_rng(n).permutation(pages)
    src, dst = order[:n], order[n: 2 * n]
    src = np.where(np.arange(n) % 3 == 2, src[0], src)  # one source may be copied many times
    for w in want:
        w[:, torch.from_numpy(dst.copy()).cuda()] = w[:, torch.from_numpy(src.copy()).cuda()]
    kv = P.paged_kv(pools[0].data_ptr(), pools[1].data_ptr(), cache, pages, page, hk, dim)
    P.copy_pages_device(kv, src, dst, layers, pools[0].stride(0))
    torch.cuda.synchronize()
    for w, p in zip(want, pools):
        assert torch.equal(w, p)


# ---- sampling

def _run_sample(x, temp=None, top_k=None, top_p=None, min_p=None, u=None, probs=True, dtype="f32", gap=0, stream=0):
    import torch
    P = pkg()
    rows, v = x.shape
    wide = torch.full((rows, v + gap), math.inf, device="cuda", dtype=_torch(dtype))
    wide[:, :v] = torch.from_numpy(x).cuda().to(_torch(dtype))
    dev = [None if a is None else torch.from_numpy(np.asarray(a, t)).cuda()
           for a, t in ((temp, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32), (u, np.float32))]
    ptr = [0 if d is None else d.data_ptr() for d in dev]
    i, k = (torch.full((rows,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    lp = torch.full((rows,), 9.0, device="cuda")
    p = torch.full((rows, v), 9.0, device="cuda") if probs else None
    torch.cuda.synchronize()
    P.sample_device(dtype, wide.data_ptr(), wide.stride(0), rows, v, ptr[4], i.data_ptr(), lp.data_ptr(), k.data_ptr(),
                    p.data_ptr() if probs else 0, *ptr[:4], stream)
    torch.cuda.synchronize()
    return (wide[:, :v].double().cpu().numpy(), i.cpu().numpy(), k.cpu().numpy(), lp.double().cpu().numpy(),
            p.double().cpu().numpy() if probs else None)


def _check_sample(x, temp=None, top_k=None, top_p=None, min_p=None, u=None, **kw):
    rows, v = x.shape
    u = np.random.default_rng(1).random(rows).astype(np.float32) if u is None else np.asarray(u, np.float32)
    x, ids, kept, lp, probs = _run_sample(x, temp, top_k, top_p, min_p, u, **kw)
    near = 0
    for r in range(rows):
        t, k = 1.0 if temp is None else float(np.float32(temp[r])), 0 if top_k is None else int(top_k[r])
        p, least = 1.0 if top_p is None else float(np.float32(top_p[r])), 0.0 if min_p is None else float(np.float32(min_p[r]))
        xr = np.where(np.isnan(x[r]), -np.inf, x[r])
        order = np.lexsort((np.arange(v), -xr))
        if xr[order[0]] == -np.inf or least > 1:
            assert (ids[r], kept[r], lp[r]) == (-1, 0, -np.inf) and (probs is None or (probs[r] == 0).all())
            continue
        if not t > 0:
            order, t = order[:1], 1.0
        elif 0 < k < v:
            order = order[:k]
        with np.errstate(invalid="ignore"):
            d = np.where(xr == xr[order[0]], 0.0, (xr - xr[order[0]]) / t)
        w = np.floor(2.0 ** 40 * np.exp(d))
        share = (np.cumsum(w[order]) - w[order]) / w[order].sum()
        unsure = False
        if p < 1:
            take = (share < p) | (np.arange(len(order)) == 0)
            unsure = bool((np.abs(share[1:] - p) < 2.0 ** -20).any())
            order = order[take]
        unsure |= bool(((np.abs(w[order] - least * 2.0 ** 40) <= 2.0 ** -21 * w[order]) & (least > 0) & (least != 1)).any())
        tail = bool(((w[order] < 4) & (w[order] > -1) & (d[order] > -40) & (d[order] < -20)).any())  # floor() near 0 or 1
        order = order[(w[order] >= least * 2.0 ** 40) & (w[order] > 0)]
        near += unsure
        if not unsure and not tail:
            assert kept[r] == len(order), (r, kept[r], len(order))
        if unsure:
            continue
        z = w[order].sum()
        run = np.zeros(v)
        run[order] = w[order] / z
        share = np.cumsum(run)
        i = ids[r]
        assert run[i] > 0, (r, i)
        assert share[i] - run[i] - 2.0 ** -20 <= u[r] <= share[i] + 2.0 ** -20, (r, i, share[i] - run[i], u[r], share[i])
        ref = d[i] - math.log(z / 2.0 ** 40)
        assert abs(lp[r] - ref) <= 2.0 ** -20 + 2.0 ** -21 * abs(d[i]), (r, lp[r], ref)
        if probs is not None:
            assert (np.abs(probs[r] - run) <= 2.0 ** -19 * run + 2.0 ** -38).all()
            assert ((probs[r] > 0) == (run > 0)).all() or tail
    assert near <= max(1, rows // 8)  # the inputs leave nearly every row decided
    return ids, kept, lp, probs


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 640, 5003, 32000, 50257])
def test_sample_against_64_bits(dtype, vocab, cuda_ok):
    rng = np.random.default_rng(vocab)
    rows = 24
    x = (2.5 * rng.standard_normal((rows, vocab))).astype(np.float32)
    x[rng.random((rows, vocab)) < 0.02] = -np.inf
    x[rng.random((rows, vocab)) < 0.01] = np.nan
    temp = rng.uniform(0.5, 1.5, rows)
    temp[::8] = 0
    top_k = np.where(rng.random(rows) < 0.5, rng.integers(1, 60, rows), 0)
    top_p = np.where(rng.random(rows) < 0.7, rng.uniform(0.05, 1, rows), 1.0)
    min_p = np.where(rng.random(rows) < 0.4, rng.uniform(0.001, 0.2, rows), 0.0)
    _check_sample(x, temp, top_k, top_p, min_p, dtype=dtype, gap=3)
    _check_sample(x, dtype=dtype, probs=False)
    _check_sample(x, temp, top_k=top_k, dtype=dtype)
    _check_sample(x, temp, top_p=top_p, dtype=dtype)
    _check_sample(x, None, min_p=min_p, dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [200, 513, 730, 1657, 4097, 20011])
def test_sample_long_lists(dtype, vocab, cuda_ok):
    """top_k around the lengths at which a list is treated in another way, in rows shorter and longer than it."""
    rng = np.random.default_rng(vocab)
    k = np.array([100, 191, 192, 193, 255, 256, 257, 300, 384, 500, 511, 512, 513, 600, 1023, 1024])
    x = (2.0 * rng.standard_normal((len(k), vocab))).astype(np.float32)
    x[3::4, ::3] = x[3::4, :1]  # many equal values, at places among the others
    temp = rng.uniform(0.5, 2.0, len(k))
    top_p = np.where(rng.random(len(k)) < 0.7, rng.uniform(0.5, 1, len(k)), 1.0)
    min_p = np.where(rng.random(len(k)) < 0.4, rng.uniform(0.001, 0.05, len(k)), 0.0)
    _check_sample(x, temp, k, dtype=dtype)
    _check_sample(x, temp, k, top_p, min_p, dtype=dtype)
    _check_sample(x, temp, None, top_p, min_p, dtype=dtype, probs=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,rows", [(100003, 5), (262144, 3), (524288, 2), (49152, 1)])
def test_sample_large_vocabularies(dtype, vocab, rows, cuda_ok):
    rng = np.random.default_rng(vocab)
    x = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    _check_sample(x, rng.uniform(0.6, 1.2, rows), None, np.full(rows, 0.9), dtype=dtype)
    _check_sample(x, rng.uniform(0.6, 1.2, rows), np.full(rows, 50000), None, np.full(rows, 0.01), dtype=dtype)
    _check_sample(x, dtype=dtype)


def test_sample_ties_go_to_the_lowest_index(cuda_ok):
    """Equal logits weigh exactly 2^40 each, so every answer is a whole number known beforehand."""
    for v in (1, 7, 1000, 40000, 300000):
        rows = 6
        x = np.zeros((rows, v), np.float32)
        x[1::2] = -0.0
        x[:, 1::2] = np.where(np.arange(v)[1::2] % 4 == 1, -0.0, 0.0)  # both zeros are one value
        k = min(v, 5)
        u = np.array([0.0, 0.25, 0.5, 0.75, 0.999, 1 - 2.0 ** -24], np.float32)
        _, ids, kept, lp, probs = _run_sample(x, top_k=np.full(rows, k), u=u)
        assert (kept == k).all() and (probs[:, :k] == np.float32(1) / np.float32(k)).all() and (probs[:, k:] == 0).all()
        assert (ids == [min(k - 1, int(float(a) * (k << 40)) >> 40) for a in u]).all()
        _, ids, kept, _, _ = _run_sample(x, temp=np.zeros(rows), u=u)
        assert (ids == 0).all() and (kept == 1).all()
        # top_p: the tokens with less than p of the weight before them
        p = np.array([0.0, 1e-9, 0.25, 0.5, 0.75, 0.9999], np.float32)
        _, ids, kept, _, _ = _run_sample(x, top_p=p, u=u)
        want = [max(1, sum(1 for i in range(v) if i < float(a) * v)) for a in p]
        assert kept.tolist() == want, (v, kept, want)
        # and after top_k, of what top_k left
        _, ids, kept, _, _ = _run_sample(x, top_k=np.full(rows, k), top_p=p, u=u)
        assert kept.tolist() == [max(1, sum(1 for i in range(k) if i < float(a) * k)) for a in p]


def test_sample_ties_at_the_boundary(cuda_ok):
    """Two levels of equal logits: the cut falls inside the lower one, and its first tokens by index stay."""
    v = 20011
    rng = np.random.default_rng(3)
    x = np.full((4, v), 1.0, np.float32)
    high = np.sort(rng.choice(v, 37, replace=False))
    x[:, high] = 3.0
    k = [37, 38, 500, 20010]
    _, ids, kept, lp, probs = _run_sample(x, top_k=k, u=[0.999] * 4)
    low = np.setdiff1d(np.arange(v), high)
    for r in range(4):
        want = np.zeros(v, bool)
        want[high] = True
        want[low[: k[r] - 37]] = True
        assert kept[r] == k[r] and ((probs[r] > 0) == want).all()
    # top_p inside the lower level too
    _check_sample(x, top_p=[0.3, 0.5, 0.9, 0.99], u=[0.1, 0.5, 0.9, 0.99])


def test_sample_strange_rows(cuda_ok):
    v = 3001
    rng = np.random.default_rng(4)
    x = rng.standard_normal((9, v)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 17] = np.inf
    x[3, [5, 900, 3000]] = np.inf
    x[4] = -np.inf
    x[4, 2999] = -3e38
    x[5] *= 1e30
    x[6] = -3.4028235e38
    x[6, 4] = 3.4028235e38
    x[7] = np.finfo(np.float32).min
    u = np.full(9, 0.5, np.float32)
    for kw in (dict(), dict(top_k=np.full(9, 40)), dict(top_p=np.full(9, 0.9)), dict(min_p=np.full(9, 0.05)), dict(temp=np.zeros(9)),
               dict(temp=np.full(9, 0.7), top_k=np.full(9, 40), top_p=np.full(9, 0.9), min_p=np.full(9, 0.05))):
        ids, kept, lp, _ = _check_sample(x, u=u, **kw)
        assert ids[0] == ids[1] == -1 and ids[2] == 17 and ids[4] == 2999 and ids[6] == 4
        assert ids[3] == (5 if "temp" in kw and kw["temp"][0] == 0 else 900)
    ids, kept, lp, probs = _check_sample(x, min_p=np.full(9, 1.5), u=u)
    assert (ids == -1).all()
    # strange settings: u outside [0, 1), tiny, negative and NaN temperatures
    _, ids, kept, lp, _ = _run_sample(x[8:9].repeat(6, 0), u=[1.0, 2.0, -1.0, np.nan, np.inf, 0.0])
    assert (ids[[0, 1, 4]] == v - 1).all() and (ids[[2, 3, 5]] == 0).all()
    _, ids, kept, lp, _ = _run_sample(x[8:9].repeat(4, 0), temp=[-1.0, np.nan, 1e-30, 1e-40], u=[0.5] * 4)
    assert (ids == x[8].argmax()).all() and (lp == 0).all()
    _, ids, kept, lp, _ = _run_sample(x[8:9].repeat(2, 0), top_p=[np.nan, -1.0], u=[0.5] * 2)
    assert (ids == x[8].argmax()).all() and (kept == 1).all()


def test_sample_shares_follow_the_distribution(cuda_ok):
    """20,000 rows of one distribution: each kept token is drawn as often as its share says (6 sigma)."""
    rng = np.random.default_rng(5)
    n, v = 20000, 50
    x = np.tile(rng.standard_normal(v).astype(np.float32) * 1.5, (n, 1))
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    _, ids, kept, _, probs = _run_sample(x, top_k=np.full(n, 20), u=u)
    count = np.bincount(ids, minlength=v)
    assert (np.abs(count - n * probs[0]) <= 6 * np.sqrt(n * probs[0] * (1 - probs[0])) + 1).all()
    assert (count[probs[0] == 0] == 0).all()


def test_sample_in_a_graph_on_a_stream(cuda_ok):
    import torch
    P = pkg()
    x = torch.randn(7, 32000, device="cuda")
    u = torch.rand(7, device="cuda")
    i = torch.empty(7, dtype=torch.int32, device="cuda")
    top_p = torch.full((7,), 0.9, device="cuda")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        P.sample_device("f32", x.data_ptr(), 32000, 7, 32000, u.data_ptr(), i.data_ptr(), top_p_ptr=top_p.data_ptr(),
                        stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        x.normal_()
        u.uniform_()
        g.replay()
        torch.cuda.synchronize()
        got = i.clone()
        P.sample_device("f32", x.data_ptr(), 32000, 7, 32000, u.data_ptr(), i.data_ptr(), top_p_ptr=top_p.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(got, i)


def test_sample_more_rows_than_run_at_once(cuda_ok):
    """Rows are begun in another order then (those without a small top_k first); each keeps its own answer."""
    rng = np.random.default_rng(8)
    rows, v = 700, 2000
    x = (2.5 * rng.standard_normal((rows, v))).astype(np.float32)
    top_k = np.where(rng.random(rows) < 0.6, rng.integers(1, 1200, rows), 0)
    temp = np.where(rng.random(rows) < 0.15, 0.0, rng.uniform(0.5, 1.5, rows))
    _check_sample(x, temp, top_k, rng.uniform(0.3, 1.05, rows))
    _check_sample(x, None, top_k)
    _check_sample(x[:, :300], temp, np.minimum(top_k, 299), None, rng.uniform(0.0, 0.1, rows))


@pytest.mark.parametrize("k", [193, 256, 300, 512, 513, 2047, 2049, 6000])
def test_sample_list_sizes(k, cuda_ok):
    """top_k around the sizes at which lists are counted, stepped through or given up, ties at the cut among them."""
    rng = np.random.default_rng(k)
    x = (2.5 * rng.standard_normal((6, 40000))).astype(np.float32)
    x[3:] = np.round(x[3:], 1)  # many equal logits
    x[5] = np.round(x[5] / 4)
    _check_sample(x, None, np.full(6, k))
    _check_sample(x, rng.uniform(0.6, 1.2, 6), np.full(6, k), rng.uniform(0.5, 0.99, 6), rng.uniform(0, 0.01, 6))
