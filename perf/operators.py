"""Cases that measure the paged-serving operators: position rotation into a paged key-value cache, attention
of one new token over it, page copies, and sampling from given random numbers.

``run`` computes an operator in its plain form (elementary torch operations) or, with ``own`` set, through
the package's entry points; ``exact`` computes the same outputs from the definitions in 64 bits.

Definitions.  A cache is a pool of pages; position p of sequence s is row p % page of page
table[s][p // page], and holds one key and one value row of each kv head.

- rope: a token's q and k heads are (where gains are given) divided by the root of their mean square plus
  eps and multiplied by the gain; their first rope_dim elements are then rotated by the angles of the
  token's position, pairs (i, i + rope_dim / 2) or, interleaved, (2 i, 2 i + 1).  q is returned, k and v
  are written into the token's cache row.
- attend: out = sum_p softmax_p(scale q . k_p) v_p over the sequence's positions p < len, query head h
  reading kv head h / (heads / kv_heads); lse = log sum_p exp(scale q . k_p).  No position: out = 0, lse = -inf.
- copy: page dst[i] of every layer becomes a copy of page src[i].
- sample: x is the row with NaN as -inf and m its maximum; a token's weight is the whole part of
  2^40 exp((x - m) (1 / T)) (T = 0: the top token alone).  By falling x, ties by rising index: the first top_k
  tokens are kept; of those, the ones with less than top_p of their weight before them; of those, the ones
  with at least min_p of the top token's weight.  With Z the kept weight and u in [0, 1), the drawn token is
  the first in index order whose running weight passes floor(u Z).  Weights are whole numbers, so sums do not
  depend on their order.
"""
import importlib
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
ONE = float(1 << 40)  # weight of the top token


def listed():
    return [
        # one sequence near the end of a 64-token prompt + 128 new tokens, PetitGPT's heads, f32 as the engine's caches
        dict(name="attend one short f32", op="attend", seqs=1, heads=9, kv_heads=3, dim=64, page=16, longest=191, act="f32",
             cache="f32", layout="head"),
        # 256 sequences of SmolLM2-135M's heads in the second half of prompt 128 + 256 new tokens
        dict(name="attend 256 ragged bf16", op="attend", seqs=256, heads=9, kv_heads=3, dim=64, page=16, longest=384, act="bf16",
             cache="bf16", layout="head"),
        # f32 activations over a bf16 cache, SmolLM2-360M's heads, lengths from none to its full context, position-major pages
        dict(name="attend 48 ragged f32 on bf16", op="attend", seqs=48, heads=15, kv_heads=5, dim=64, page=32, longest=2048,
             act="f32", cache="bf16", layout="pos"),
        # three long documents: many pages, few rows, so the length itself has to be split
        dict(name="attend 3 long f16", op="attend", seqs=3, heads=32, kv_heads=8, dim=128, page=64, longest=100003, act="f16",
             cache="f16", layout="head"),
        # the position step of a single-sequence decode
        dict(name="rope one token f32", op="rope", seqs=1, new=1, heads=9, kv_heads=3, dim=64, page=16, longest=192, act="f32",
             cache="f32", layout="head", rope_dim=64, interleaved=False, norm=False),
        # one new token of 256 sequences, with normed queries and keys
        dict(name="rope 256 tokens normed bf16", op="rope", seqs=256, new=1, heads=9, kv_heads=3, dim=64, page=16, longest=384,
             act="bf16", cache="bf16", layout="head", rope_dim=64, interleaved=False, norm=True),
        # the prompts of 24 sequences in one pass: f32 activations into a bf16 cache, part of the head rotated, pairs adjacent
        dict(name="rope prompts f32 into bf16", op="rope", seqs=24, new=1021, heads=15, kv_heads=5, dim=64, page=32, longest=2048,
             act="f32", cache="bf16", layout="pos", rope_dim=48, interleaved=True, norm=True),
        # a fork that is about to be written: the last page of one sequence, in every layer
        dict(name="copy one page", op="copy", layers=30, pages=64, kv_heads=3, dim=64, page=16, moves=1, cache="f32"),
        # compaction of a fragmented pool: 1,500 pages of every layer
        dict(name="copy 1500 pages", op="copy", layers=30, pages=4096, kv_heads=5, dim=64, page=32, moves=1500, cache="bf16"),
        # the one row of a single-sequence decode, SmolLM2's vocabulary
        dict(name="sample one row f32", op="sample", rows=1, vocab=49152, dtype="f32", probs=False, plain=False),
        # a batch whose requests each bring their own settings, greedy ones among them
        dict(name="sample 256 rows f32", op="sample", rows=256, vocab=49152, dtype="f32", probs=False, plain=False),
        # GPT-2's odd vocabulary in bf16, temperature and top-p only, with the distribution that a draft check needs
        dict(name="sample 33 rows bf16 probs", op="sample", rows=33, vocab=50257, dtype="bf16", probs=True, plain=True),
    ]


def spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "rope", "copy", "sample"])
    kv = rng.choice([1, 2, 3, 4, 5, 8, 12])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    layout = rng.choice(["head", "pos"])
    act, cache = rng.choice([("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f16")])
    if op == "attend":
        longest = spread(rng, 1, 131072)
        room = 2.0e8 / (longest * kv * dim)  # positions x kv heads x head_dim stay below the largest listed case's
        if room < 1:
            longest, room = max(1, int(longest * room)), 1
        seqs = spread(rng, 1, max(1, min(512, int(room))))
        return dict(op=op, seqs=seqs, heads=kv * rng.choice([1, 2, 3, 4, 5, 8, 16]), kv_heads=kv, dim=dim, page=page,
                    longest=longest, act=act, cache=cache, layout=layout)
    if op == "rope":
        new = spread(rng, 1, 2048)
        seqs = spread(rng, 1, max(1, 24576 // new))
        heads = kv * rng.choice([1, 2, 3, 4, 5])
        while seqs * new * heads * dim > 2.3e7 and seqs > 1:
            seqs = (seqs + 1) // 2
        while seqs * new * heads * dim > 2.3e7:
            new = (new + 1) // 2
        return dict(op=op, seqs=seqs, new=new, heads=heads, kv_heads=kv, dim=dim, page=page, longest=new + spread(rng, 1, 1024),
                    act=act, cache=cache, layout=layout, rope_dim=rng.choice([dim, dim, dim // 2, 0]),
                    interleaved=rng.random() < 0.4, norm=rng.random() < 0.5)
    if op == "copy":
        cache = rng.choice(["f32", "f16", "bf16"])
        layers = rng.choice([1, 2, 12, 30, 32])
        per = layers * kv * dim * page * BYTES[cache] * 2
        pages = max(4, min(4096, int(2.5e9 / per)))
        return dict(op=op, layers=layers, pages=pages, kv_heads=kv, dim=dim, page=page,
                    moves=spread(rng, 1, max(1, min(pages // 2, int(9e8 / per)))), cache=cache)
    vocab = spread(rng, 500, 262144)
    return dict(op="sample", rows=spread(rng, 1, max(1, min(512, int(1.2e7 / vocab)))), vocab=vocab,
                dtype=rng.choice(["f32", "f16", "bf16"]), probs=rng.random() < 0.3, plain=rng.random() < 0.3)


def lengths(c):
    """Cache lengths by sequence: the first is the longest, the others spread over the rest, every eleventh sequence new."""
    n = np.arange(c["seqs"])
    if c["op"] == "rope":  # every sequence gets `new` tokens after what it holds
        return c["longest"] - (np.modf(n * 0.6180339887)[0] * (c["longest"] - c["new"])).astype(np.int64)
    got = c["longest"] - (np.modf(n * 0.6180339887)[0] * c["longest"] * (0.66 if c["longest"] <= 384 else 0.98)).astype(np.int64)
    got[n % 11 == 10] = 0
    return got


def pool(c, gen, n_pages, layers=None):
    """Key and value pages of normal values, [page][kv head][position][dim] or [page][position][kv head][dim]."""
    shape = [n_pages, c["kv_heads"], c["page"], c["dim"]]
    if c.get("layout") == "pos":
        shape = [n_pages, c["page"], c["kv_heads"], c["dim"]]
    if layers:
        shape = [layers] + shape
    return [torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if c["cache"] == "f32" else TYPES[c["cache"]])
            for _ in range(2)]


def strides(c):
    """Elements between pages, kv heads and positions."""
    d, h, p = c["dim"], c["kv_heads"], c["page"]
    return (h * p * d, d, h * d) if c.get("layout") == "pos" else (h * p * d, p * d, d)


def tables(c, gen, lens):
    """Every sequence's pages, drawn from all over the pool; -1 past a sequence's last page."""
    need = -(-lens // c["page"])
    most = max(1, int(need.max()))
    n_pages = int(need.sum()) + max(4, int(need.sum()) // 8)
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    used = torch.arange(most)[None, :] < torch.from_numpy(need)[:, None]
    table = torch.full((c["seqs"], most), -1, dtype=torch.int32, device="cuda")
    table[used.cuda()] = order[: int(need.sum())]
    return table, n_pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, {"case": case}
    if c["op"] in ("attend", "rope"):
        lens = lengths(c)
        s["table"], s["n_pages"] = tables(c, gen, lens)
        s["k"], s["v"] = pool(c, gen, s["n_pages"])
        s["len"] = torch.from_numpy(lens.astype(np.int32)).cuda()
    if c["op"] == "attend":
        s["q"] = torch.randn(c["seqs"], c["heads"], c["dim"], generator=gen, device="cuda").to(TYPES[c["act"]])
        s["scale"] = c["dim"] ** -0.5
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(c["seqs"], c["heads"], device="cuda")
    elif c["op"] == "rope":
        n = c["seqs"] * c["new"]
        s["qkv"] = torch.randn(n, (c["heads"] + 2 * c["kv_heads"]) * c["dim"], generator=gen, device="cuda").to(TYPES[c["act"]])
        s["seq"] = torch.arange(c["seqs"], device="cuda", dtype=torch.int32).repeat_interleave(c["new"])
        s["pos"] = (torch.from_numpy(lens).cuda()[:, None] - c["new"] + torch.arange(c["new"], device="cuda")).reshape(-1).to(torch.int32)
        half = c["rope_dim"] // 2
        inv = torch.from_numpy(10000.0 ** (-np.arange(half) / max(1, half))).cuda()
        angle = torch.arange(c["longest"], device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        s["q_gain"], s["k_gain"] = (1 + 0.1 * torch.randn(c["dim"], generator=gen, device="cuda") for _ in range(2)) if c["norm"] else (None, None)
        s["q"] = torch.empty(n, c["heads"], c["dim"], device="cuda", dtype=TYPES[c["act"]])
    elif c["op"] == "copy":
        s["n_pages"] = c["pages"]
        s["k"], s["v"] = pool(c, gen, c["pages"], c["layers"])
        order = np.random.default_rng(seed).permutation(c["pages"]).astype(np.int32)
        s["src"], s["dst"] = order[: c["moves"]].copy(), order[c["moves"]: 2 * c["moves"]].copy()
    else:
        r, v = c["rows"], c["vocab"]
        x = 2.5 * torch.randn(r, v, generator=gen, device="cuda")
        x += 6.0 * (torch.rand(r, v, generator=gen, device="cuda") < 3e-4)  # the few likely tokens
        x[torch.rand(r, v, generator=gen, device="cuda") < 0.01] = -math.inf  # tokens that a grammar bans
        s["logits"] = x.to(TYPES[c["dtype"]])
        rng = np.random.default_rng(seed)
        temp, top_p = rng.uniform(0.6, 1.2, r), rng.uniform(0.8, 1.0, r)
        top_k, min_p = np.zeros(r), np.zeros(r)
        if not c["plain"]:
            top_k = np.where(rng.random(r) < 0.7, np.exp(rng.uniform(0, math.log(1000), r)), 0)
            min_p = np.where(rng.random(r) < 0.4, rng.uniform(0.01, 0.1, r), 0)
            temp[rng.random(r) < 0.1] = 0
            top_p[rng.random(r) < 0.2] = 1
            if r == 1:
                temp[0], top_k[0], top_p[0], min_p[0] = 0.8, 40, 0.95, 0.0
        for name, a, t in (("temp", temp, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                           ("min_p", min_p, torch.float32)):
            s[name] = torch.from_numpy(a).to(t).cuda()
        s["u"] = torch.rand(r, generator=gen, device="cuda")
        s["id"], s["kept"] = (torch.empty(r, dtype=torch.int32, device="cuda") for _ in range(2))
        s["logprob"] = torch.empty(r, device="cuda")
        s["p"] = torch.empty(r, v, device="cuda") if c["probs"] else None
    if own:  # what the program keeps beside its tensors: the cache's descriptor and the attention's workspace
        s["lib"] = lib = importlib.import_module("microllm-lab_b200")
        if c["op"] != "sample":
            s["kv"] = lib.paged_kv(s["k"].data_ptr(), s["v"].data_ptr(), c["cache"], s["n_pages"], c["page"], c["kv_heads"], c["dim"],
                                   strides(c))
        if c["op"] == "attend":
            s["ws"] = torch.zeros(lib.paged_attn_workspace(c["seqs"], c["heads"], c["dim"]), dtype=torch.uint8, device="cuda")
    return s


def run(s):
    c = s["case"]
    return (OWN if own else PLAIN)[c["op"]](s, c)


# ---- through the package's entry points

def own_attend(s, c):
    q, out = s["q"], s["out"]
    s["lib"].paged_attn_device(s["kv"], c["act"], q.data_ptr(), q.stride(0), c["seqs"], c["heads"], s["len"].data_ptr(),
                               s["table"].data_ptr(), s["table"].stride(0), s["scale"], out.data_ptr(), out.stride(0),
                               s["ws"].data_ptr(), s["ws"].numel(), s["lse"].data_ptr())
    return out, s["lse"]


def own_rope(s, c):
    qkv, q = s["qkv"], s["q"]
    gains = (s["q_gain"].data_ptr(), s["k_gain"].data_ptr()) if c["norm"] else (0, 0)
    s["lib"].rope_append_device(s["kv"], c["act"], qkv.data_ptr(), qkv.stride(0), qkv.shape[0], c["heads"], s["seq"].data_ptr(),
                                s["pos"].data_ptr(), s["table"].data_ptr(), c["seqs"], s["table"].stride(0), s["cos"].data_ptr(),
                                s["sin"].data_ptr(), c["longest"], c["rope_dim"], q.data_ptr(), q.stride(0), c["interleaved"],
                                *gains, EPS)
    return q, s["k"], s["v"]


def own_copy(s, c):
    s["lib"].copy_pages_device(s["kv"], s["src"], s["dst"], c["layers"], s["k"].stride(0))
    return s["k"], s["v"]


def own_sample(s, c):
    x = s["logits"]
    s["lib"].sample_device(c["dtype"], x.data_ptr(), x.stride(0), c["rows"], c["vocab"], s["u"].data_ptr(), s["id"].data_ptr(),
                           s["logprob"].data_ptr(), s["kept"].data_ptr(), s["p"].data_ptr() if c["probs"] else 0,
                           s["temp"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr())
    return [s["id"], s["kept"], s["logprob"]] + ([s["p"]] if c["probs"] else [])


# ---- plain forms

def plain_attend(s, c):
    """The sequences' rows gathered to the longest length, then two batched products around a masked softmax."""
    b, hk, d = c["seqs"], c["kv_heads"], c["dim"]
    table = s["table"].clamp(min=0).long()
    span = table.shape[1] * c["page"]
    live = torch.arange(span, device="cuda")[None, :] < s["len"][:, None]
    rows = [t[table] if c["layout"] == "pos" else t[table].transpose(2, 3) for t in (s["k"], s["v"])]
    k, v = (t.reshape(b, span, hk, d).float().permute(0, 2, 1, 3) for t in rows)
    v = v.masked_fill(~live[:, None, :, None], 0.0)
    q = s["q"].float().reshape(b, hk, c["heads"] // hk, d)
    x = (q @ k.transpose(2, 3) * s["scale"]).masked_fill(~live[:, None, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m > -math.inf, m, torch.zeros_like(m))
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    out = (e @ v) / torch.where(z > 0, z, torch.ones_like(z))
    lse = m + z.log()
    s["out"].copy_(out.reshape(b, c["heads"], d))
    s["lse"].copy_(lse.reshape(b, c["heads"]))
    return s["out"], s["lse"]


def plain_turn(x, gain, cos, sin, c):
    """x [tokens][heads][dim] in f32: normed where there is a gain, then its first rope_dim elements turned."""
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * gain
    r = c["rope_dim"]
    head, rest = x[..., :r], x[..., r:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if c["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., : r // 2], head[..., r // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def plain_rope(s, c):
    n, h, hk, d = s["qkv"].shape[0], c["heads"], c["kv_heads"], c["dim"]
    q, k, v = s["qkv"].float().reshape(n, h + 2 * hk, d).split([h, hk, hk], 1)
    pos = s["pos"].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    s["q"].copy_(plain_turn(q, s["q_gain"], cos, sin, c))
    k = plain_turn(k, s["k_gain"], cos, sin, c)
    page, at = s["table"][s["seq"].long(), pos // c["page"]].long(), pos % c["page"]
    k, v = k.to(s["k"].dtype), v.to(s["v"].dtype)
    if c["layout"] == "pos":
        s["k"][page, at], s["v"][page, at] = k, v
    else:
        s["k"][page, :, at], s["v"][page, :, at] = k, v
    return s["q"], s["k"], s["v"]


def plain_copy(s, c):
    src, dst = torch.from_numpy(s["src"]).long().cuda(), torch.from_numpy(s["dst"]).long().cuda()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return s["k"], s["v"]


def plain_sample(s, c):
    x = s["logits"].float()
    x = x.masked_fill(x.isnan(), -math.inf)
    r, n = x.shape
    temp, greedy = s["temp"][:, None], ~(s["temp"][:, None] > 0)
    m = x.amax(-1, keepdim=True)
    d = torch.where(x == m, 0.0, (x - m) * torch.where(greedy, 1.0, 1.0 / temp))
    w = torch.where(x > -math.inf, d.exp() * ONE, 0.0).to(torch.int64)
    order = x.argsort(dim=-1, descending=True, stable=True)
    rank = torch.arange(n, device="cuda")[None, :]
    k = s["top_k"].long()[:, None]
    k = torch.where(greedy, 1, torch.where((k <= 0) | (k > n), n, k))
    sorted_w = torch.where(rank < k, w.gather(-1, order), 0)
    total = sorted_w.sum(-1, keepdim=True)
    before = (sorted_w.cumsum(-1) - sorted_w).double()
    enough = (before < s["top_p"].double()[:, None] * total.double()) | (s["top_p"][:, None] >= 1) | (rank == 0)
    keep = enough & (sorted_w > 0) & (sorted_w.double() >= s["min_p"].double()[:, None] * ONE)
    kept_w = torch.where(torch.zeros_like(keep).scatter(-1, order, keep), w, 0)
    running = kept_w.cumsum(-1)
    z = running[:, -1:]
    aim = torch.minimum((s["u"].double()[:, None] * z.double()).floor().to(torch.int64), z - 1)
    at = (running <= aim).sum(-1, keepdim=True)
    none = z == 0  # every token banned
    share = z.double().float() / ONE
    s["id"].copy_(torch.where(none, -1, at)[:, 0])
    s["kept"].copy_(keep.sum(-1))
    s["logprob"].copy_(torch.where(none, -math.inf, d.gather(-1, at.clamp(max=n - 1)) - share.log())[:, 0])
    out = [s["id"], s["kept"], s["logprob"]]
    if c["probs"]:
        s["p"].copy_(torch.where(none, 0.0, kept_w.float() / z.float()))
        out.append(s["p"])
    return out


OWN = {"attend": own_attend, "rope": own_rope, "copy": own_copy, "sample": own_sample}
PLAIN = {"attend": plain_attend, "rope": plain_rope, "copy": plain_copy, "sample": plain_sample}


# ---- from the definitions in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "copy":
        k, v = s["k"].clone(), s["v"].clone()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            k[:, b], v[:, b] = s["k"][:, a], s["v"][:, a]
        return k, v
    if c["op"] == "attend":
        out, lse = [], []
        rep = c["heads"] // c["kv_heads"]
        for i, n in enumerate(s["len"].tolist()):
            if n == 0:
                out.append(torch.zeros(c["heads"], c["dim"], dtype=torch.float64, device="cuda"))
                lse.append(torch.full((c["heads"],), -math.inf, dtype=torch.float64, device="cuda"))
                continue
            at = torch.arange(n, device="cuda")
            page, row = s["table"][i, at // c["page"]].long(), at % c["page"]
            rows = []
            for t in (s["k"], s["v"]):
                t = t[page, row] if c["layout"] == "pos" else t[page, :, row]
                rows.append(t.double())  # [n][kv head][dim]
            q = s["q"][i].double().reshape(c["kv_heads"], rep, c["dim"])
            x = s["scale"] * torch.bmm(q, rows[0].permute(1, 2, 0))  # [kv head][query head of it][n]
            l = torch.logsumexp(x, -1)
            out.append(torch.bmm((x - l[..., None]).exp(), rows[1].transpose(0, 1)).reshape(c["heads"], c["dim"]))
            lse.append(l.reshape(-1))
        return torch.stack(out), torch.stack(lse)
    if c["op"] == "rope":
        n, hk, d, r = s["qkv"].shape[0], c["kv_heads"], c["dim"], c["rope_dim"]
        x = s["qkv"].double().reshape(n, -1, d)
        pos = s["pos"].long()
        gains = [(0, c["heads"], s["q_gain"]), (c["heads"], c["heads"] + hk, s["k_gain"])]
        turned = []
        for lo, hi, gain in gains:
            y = x[:, lo:hi]
            if gain is not None:
                y = y * gain.double() / torch.sqrt((y * y).sum(-1, keepdim=True) / d + EPS)
            z = y.clone()
            for i in range(r // 2):
                a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + r // 2)
                co, si = s["cos"][pos, i].double()[:, None], s["sin"][pos, i].double()[:, None]
                z[..., a] = y[..., a] * co - y[..., b] * si
                z[..., b] = y[..., a] * si + y[..., b] * co
            turned.append(z)
        k, v = s["k"].double(), s["v"].double()
        page, at = s["table"][s["seq"].long(), pos // c["page"]].long(), pos % c["page"]
        for h in range(hk):
            where = (page, at, h) if c["layout"] == "pos" else (page, h, at)
            k[where] = turned[1][:, h]
            v[where] = x[:, c["heads"] + hk + h]
        return turned[0], k, v
    # sample: row by row in numpy; ids and counts hang on the rounding of the weights, so they have no 64-bit value of their own
    logprob, probs, torn = [], [], False
    x_all = s["logits"].double().cpu().numpy()
    par = {n: s[n].double().cpu().numpy() for n in ("temp", "top_p", "min_p", "u")}
    top_k = s["top_k"].cpu().numpy()
    for i, x in enumerate(x_all):
        t = par["temp"][i]
        p = np.zeros(len(x))
        order = np.lexsort((np.arange(len(x)), -x))
        if t > 0:
            order = order[: top_k[i] if 0 < top_k[i] < len(x) else len(x)]
        else:
            order, t = order[:1], 1.0
        d = (x - x.max()) * float(np.float32(1) / np.float32(t))
        w = np.exp(d)
        before = np.cumsum(w[order]) - w[order]
        if par["top_p"][i] < 1:
            order = order[(before < par["top_p"][i] * w[order].sum()) | (np.arange(len(order)) == 0)]
        order = order[w[order] >= par["min_p"][i]]
        order = order[w[order] >= 1 / ONE]
        p[order] = w[order] / w[order].sum()
        running = np.cumsum(p)
        at = min(int(np.searchsorted(running, par["u"][i], side="right")), int(order.max()))
        # u this near to a step between two tokens: 32-bit weights decide which of them it is
        torn |= len(order) > 1 and bool((np.abs(running[np.sort(order)[:-1]] - par["u"][i]) < 3e-7).any())
        logprob.append(d[at] - math.log(w[order].sum()))
        probs.append(p)
    if torn and not c["probs"]:
        return None
    out = [None, None, None if torn else torch.tensor(logprob, dtype=torch.float64)]
    return out + [torch.from_numpy(np.stack(probs))] if c["probs"] else out


def work(case):
    """Bytes that have to be read and written once, and the operations of the two products (others count by element)."""
    c = case
    if c["op"] == "copy":
        return {"bytes": 2.0 * 2 * c["moves"] * c["layers"] * c["kv_heads"] * c["page"] * c["dim"] * BYTES[c["cache"]], "flops": 0.0}
    if c["op"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": float(n * BYTES[c["dtype"]] + (4 * n if c["probs"] else 0) + 32 * c["rows"]), "flops": 4.0 * n}
    lens = lengths(c)
    if c["op"] == "attend":
        kv = float(lens.sum()) * c["kv_heads"] * c["dim"]
        rows = c["seqs"] * c["heads"]
        pages = float((-(-lens // c["page"])).sum())
        return {"bytes": 2 * kv * BYTES[c["cache"]] + rows * (2 * c["dim"] * BYTES[c["act"]] + 4) + 4 * (pages + c["seqs"]),
                "flops": 4.0 * float(lens.sum()) * c["heads"] * c["dim"]}
    n = c["seqs"] * c["new"]
    table = 4.0 * c["rope_dim"] * min(n, c["longest"])  # cos and sin of the positions in use
    return {"bytes": n * c["dim"] * ((2 * c["heads"] + 2 * c["kv_heads"]) * BYTES[c["act"]] + 2 * c["kv_heads"] * BYTES[c["cache"]])
            + 12.0 * n + table, "flops": n * c["dim"] * (c["heads"] + c["kv_heads"]) * (7.0 if c["norm"] else 3.0)}
