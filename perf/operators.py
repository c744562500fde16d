"""The 4-bit latent cache's operators as a user calls them, beside their plain forms in torch.

Five kinds of case, all over pages of 64 tokens named by a block table:

  append   mla_prep (a layer's append) into the 4-bit cache, and the lift of what the call's sequences hold
  attn     attention of a packed call's rows over their sequences' whole 4-bit cache, causal among the fresh rows
  picks    the same over the 2048 slots an indexer picked for each row
  weights  every cached token's attention weight, summed over heads and rows, added to its running sum
  evict    the plan of which tokens leave a sequence's cache, and the move of the survivors

The latent row is 416 bytes: 512 e2m1 codes (value 2j in the low nibble of byte j), 32 e4m3 scales (one per
16 values, amax / 6), 64 bf16 roped key dims.
"""
import random

import numpy as np
import torch

own = False

PAGE, LAT, PE, ROW = 64, 512, 64, 416
QL, DIM, TOPK = 2048, LAT + PE, 2048
IDX_PAGE = PAGE * 132
WORKSPACE = 40 << 20   # the attention's workspace: two partial row tiles an SM
SCALE = 256 ** -0.5    # the score scale of 192 + 64 dims a head
DEV = "cuda"


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # a decode step of eight sequences: one fresh row each
        {"name": "append_step", "kind": "append", "nseq": 8, "fresh": 8, "prefix": 300, "full": False},
        # a packed prefill chunk of an indexer layer, ragged sequences
        {"name": "append_chunk", "kind": "append", "nseq": 16, "fresh": 16384, "prefix": 2048, "full": True},
        # one short sequence, one token: latency
        {"name": "attn_one", "kind": "attn", "nseq": 1, "ctx": 777, "qlen": 1, "heads": 64, "ragged": False},
        # a serving batch: ragged contexts, two tokens a sequence (one drafted)
        {"name": "attn_batch", "kind": "attn", "nseq": 32, "ctx": 8192, "qlen": 2, "heads": 64, "ragged": True},
        # one long context split over the whole GPU
        {"name": "attn_long", "kind": "attn", "nseq": 2, "ctx": 262144, "qlen": 1, "heads": 128, "ragged": True},
        # the indexer's picks of a small decode batch with an odd number of heads, some contexts below 2048
        {"name": "picks_step", "kind": "picks", "nseq": 8, "ctx": 3000, "qlen": 1, "heads": 40, "ragged": True},
        # a chunk of rows, each with its own 2048 picks
        {"name": "picks_chunk", "kind": "picks", "nseq": 4, "ctx": 16384, "qlen": 128, "heads": 64, "ragged": True},
        # weights of a small batch and of the serving batch
        {"name": "weights_step", "kind": "weights", "nseq": 4, "ctx": 1000, "qlen": 1, "heads": 64, "ragged": True},
        {"name": "weights_batch", "kind": "weights", "nseq": 32, "ctx": 8192, "qlen": 1, "heads": 64, "ragged": True},
        # a step that drops the few tokens over the budget
        {"name": "evict_step", "kind": "evict", "nseq": 8, "ctx": 1088, "budget": 1024, "sink": 4, "recent": 128},
        # a serving batch cut to half its cache
        {"name": "evict_batch", "kind": "evict", "nseq": 48, "ctx": 16384, "budget": 8000, "sink": 4, "recent": 512},
        # one very long sequence
        {"name": "evict_long", "kind": "evict", "nseq": 1, "ctx": 1000000, "budget": 262144, "sink": 16,
         "recent": 4096},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["append", "attn", "attn", "picks", "weights", "evict"])
    if kind == "append":
        fresh = _log(rng, 1, 16384)
        return {"kind": kind, "nseq": min(fresh, rng.randint(1, 16)), "fresh": fresh, "prefix": rng.randint(0, 2048),
                "full": rng.random() < 0.5}
    if kind == "evict":
        nseq = _log(rng, 1, 48)
        ctx = _log(rng, 65, min(1000000, 786432 // nseq))
        budget = max(1, int(ctx * rng.uniform(0.2, 1.05)))
        sink = rng.randint(0, min(16, budget))
        return {"kind": kind, "nseq": nseq, "ctx": ctx, "budget": budget, "sink": sink,
                "recent": rng.randint(0, budget - sink)}
    heads = rng.choice([1, 8, 16, 24, 40, 64, 128])
    if kind == "picks":
        nseq, qlen = rng.randint(1, 4), _log(rng, 1, 48)
        return {"kind": kind, "nseq": nseq, "ctx": _log(rng, 1, 32768), "qlen": qlen, "heads": heads, "ragged": True}
    nseq, qlen = _log(rng, 1, 64), rng.randint(1, 4)
    return {"kind": kind, "nseq": nseq, "ctx": _log(rng, 1, 262144 // (nseq * qlen)), "qlen": qlen, "heads": heads,
            "ragged": rng.random() < 0.7}


def _shape(case):
    """The call's (prefix lengths, fresh rows) by sequence: the case's own, the same for every seed."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["nseq"]
    if case["kind"] == "append":
        cuts = sorted(r.sample(range(1, case["fresh"]), n - 1)) if n > 1 else []
        fresh = [b - a for a, b in zip([0] + cuts, cuts + [case["fresh"]])]
        return [r.randint(0, case["prefix"]) for _ in range(n)], fresh
    if case["kind"] == "evict":
        return [max(1, int(case["ctx"] * (1 if n == 1 else r.uniform(0.8, 1)))) for _ in range(n)], [0] * n
    q = case["qlen"]
    ctx = [int(case["ctx"] * r.uniform(0.3, 1)) if case["ragged"] else case["ctx"] for _ in range(n)]
    return [max(0, c - q) for c in ctx], [q] * n


# ------------------------------------------------------------------------------------------ the format

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _quant(v):
    """[n, 512] f32 -> e2m1 codes [n, 256] u8 and e4m3 scales [n, 32] u8."""
    g = v.reshape(-1, 32, 16)
    s = (g.abs().amax(-1) / 6).clamp(max=448.0).to(torch.float8_e4m3fn)
    sf = s.float()[..., None]
    y = torch.where(sf > 0, g / sf, torch.zeros_like(g))
    a = y.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i in range(7):  # between codes i and i + 1: the midpoint goes to the even code
        mid = (GRID[i] + GRID[i + 1]) / 2
        code += ((a >= mid) if i % 2 else (a > mid)).to(torch.uint8)
    code |= (torch.signbit(y) & (sf > 0)).to(torch.uint8) << 3
    code = code.reshape(-1, 256, 2)
    return code[..., 0] | (code[..., 1] << 4), s.view(torch.uint8)


def _rows(lat, pe):
    """Cache rows [n, 416] u8 of latent rows and roped key dims."""
    codes, s = _quant(lat.float())
    return torch.cat([codes, s, pe.contiguous().view(torch.uint8).reshape(-1, 128)], 1)


def _lift(rows):
    """[n, 416] u8 -> [n, 576] f32."""
    lut = torch.tensor(GRID + [-x for x in GRID], device=rows.device)
    codes = rows[:, :256]
    v = lut[torch.stack([codes & 15, codes >> 4], -1).long()].reshape(-1, 32, 16)
    v = v * rows[:, 256:288].contiguous().view(torch.float8_e4m3fn).float()[..., None]
    return torch.cat([v.reshape(-1, LAT), rows[:, 288:].contiguous().view(torch.bfloat16).float()], 1)


# ------------------------------------------------------------------------------------------ inputs

def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _cache(g, n_pages):
    """A pool of 4-bit rows as an append leaves it: normed latents, roped key dims."""
    n = n_pages * PAGE
    out = torch.empty(n, ROW, dtype=torch.uint8, device=DEV)
    for a in range(0, n, 1 << 17):
        b = min(n, a + (1 << 17))
        out[a:b] = _rows(_normal(g, b - a, LAT), _normal(g, b - a, PE))
    return out


def prepare(case, seed):
    case = dict(case)
    prefix, fresh = _shape(case)
    lens = [p + f for p, f in zip(prefix, fresh)]
    if case["kind"] == "append":  # the lift covers what the append wrote: whole sequences of fresh rows
        lens = list(fresh)
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages = [-(-n // PAGE) for n in lens]
    n_pages, max_pages = max(1, sum(pages)), max(1, *pages)
    perm = np.random.default_rng(seed).permutation(n_pages).astype(np.int32)
    bt = np.full((len(lens), max_pages), -1, np.int32)
    at = 0
    for i, n in enumerate(pages):
        bt[i, :n] = perm[at:at + n]
        at += n
    T = sum(fresh)
    cu = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int64)
    to = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(DEV)
    s = {"kind": case["kind"], "nseq": len(lens), "n_pages": n_pages, "max_pages": max_pages, "bt": to(bt), "T": T,
         "cu": to(cu), "lens": to(np.array(lens, np.int32)), "top": max(lens), "ctx": sum(lens)}
    if case["kind"] == "append":
        pos = np.concatenate([p + np.arange(f) for p, f in zip(prefix, fresh)])
        rel = np.concatenate([np.arange(f) for f in fresh])
        seq = np.repeat(np.arange(len(lens)), fresh)
        s |= {"full": case["full"], "x": _normal(g, T, QL + DIM + (128 if case["full"] else 0)),
              "g_q": (1 + 0.1 * _normal(g, QL)), "g_kv": (1 + 0.1 * _normal(g, LAT)),
              "ik_w": (1 + 0.1 * _normal(g, 128)), "ik_b": 0.1 * _normal(g, 128),
              "pos": to(pos.astype(np.int32)), "slot": to((bt[seq, rel // PAGE].astype(np.int64) * PAGE + rel % PAGE)),
              "kv": torch.zeros(n_pages * PAGE, ROW, dtype=torch.uint8, device=DEV),
              "idx": torch.zeros(n_pages * IDX_PAGE, dtype=torch.uint8, device=DEV),
              "qq": torch.zeros(T, QL, dtype=torch.uint8, device=DEV),
              "qsf": torch.zeros(4, T, dtype=torch.int32, device=DEV),
              "kvd": torch.zeros(sum(lens), DIM, dtype=torch.bfloat16, device=DEV)}
        ang = torch.arange(int(pos.max()) + 1, dtype=torch.float64)[:, None] * \
            (8e6 ** (-torch.arange(32, dtype=torch.float64) / 32))
        s["rope"] = torch.cat([ang.cos(), ang.sin()], 1).to(torch.bfloat16).to(DEV)
        return s
    if case["kind"] == "evict":
        n = n_pages * PAGE
        acc = torch.exp(2 * torch.randn(n, generator=g, device=DEV))
        acc[torch.rand(n, generator=g, device=DEV) < 0.1] = 0  # tokens nothing has attended to yet
        pos = np.zeros(n, np.int32)
        for i, m in enumerate(lens):
            j = np.arange(m)
            pos[bt[i, j // PAGE].astype(np.int64) * PAGE + j % PAGE] = j
        s |= {"acc": acc, "pos": to(pos), "seen": s["lens"].clone(), "budget": case["budget"], "sink": case["sink"],
              "recent": case["recent"],
              "kv": torch.randint(0, 256, (n, ROW), dtype=torch.uint8, device=DEV, generator=g),
              "moves": torch.full((len(lens), case["budget"], 2), -1, dtype=torch.int32, device=DEV),
              "n_moves": torch.zeros(len(lens), dtype=torch.int32, device=DEV),
              "new_lens": torch.zeros(len(lens), dtype=torch.int32, device=DEV)}
        return s
    H = case["heads"]
    s |= {"H": H, "q": _normal(g, T, H, DIM, std=1.2), "kv": _cache(g, n_pages), "qmax": max(fresh),
          "out": torch.zeros(T, H, LAT, dtype=torch.bfloat16, device=DEV),
          "lse": torch.zeros(T, H, dtype=torch.float32, device=DEV),
          "ws": torch.empty(WORKSPACE, dtype=torch.uint8, device=DEV)}
    if case["kind"] == "weights":
        s["acc"] = torch.rand(n_pages * PAGE, generator=g, device=DEV)
        s["lse"] = torch.logsumexp(_scores(s)[0], -1)  # what the attention of the same rows left
    if case["kind"] == "picks":
        ind = np.full((T, TOPK), -1, np.int32)
        rng = np.random.default_rng(seed + 1)
        tlen, r = np.zeros(T, np.int32), 0
        for i, (p, f) in enumerate(zip(prefix, fresh)):
            for t in range(f):
                keys = p + t + 1
                pick = np.arange(keys) if keys <= TOPK else np.sort(rng.choice(keys, TOPK, replace=False))
                ind[r, :len(pick)] = bt[i, pick // PAGE] * PAGE + pick % PAGE
                tlen[r] = len(pick)
                r += 1
        s |= {"ind": to(ind), "tlen": to(tlen)}
    return s


# ------------------------------------------------------------------------------------------ the plain forms

def _slots(s):
    """Slots [nseq, longest] of every sequence's tokens and which of them exist."""
    j = torch.arange(s["top"], device=DEV)
    ok = j[None] < s["lens"][:, None]
    return torch.where(ok, s["bt"][:, j // PAGE].long() * PAGE + j % PAGE, 0), ok


def _padded_rows(s):
    """Row of q [nseq, longest fresh] and which of them exist."""
    t = torch.arange(s["qmax"], device=DEV)
    n = (s["cu"][1:] - s["cu"][:-1])[:, None]
    return torch.where(t[None] < n, s["cu"][:-1, None] + t, 0), t[None] < n, n


def _scores(s):
    """Scores [nseq rows of q, heads, longest] f32 with -inf where a row may not look, the keys they are with."""
    slots, ok = _slots(s)
    k = _lift(s["kv"][slots.reshape(-1)]).reshape(s["nseq"], s["top"], DIM)
    rows, live, n = _padded_rows(s)
    q = s["q"][rows].float().reshape(s["nseq"], -1, DIM)
    x = torch.bmm(q, k.transpose(1, 2)).reshape(s["nseq"], s["qmax"], s["H"], -1) * SCALE
    last = (s["lens"][:, None] - n + torch.arange(s["qmax"], device=DEV))  # the last key a row sees
    seen = ok[:, None] & (torch.arange(s["top"], device=DEV) <= last[..., None])
    x = torch.where(seen[:, :, None], x, -torch.inf)
    return x[live], k, live, slots, ok


def _softmax(x):
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(x - m)
    l = e.sum(-1, keepdim=True)
    return e / torch.where(l > 0, l, torch.ones_like(l)), (m + torch.log(l))[..., 0]


def _index(s):
    """The indexer cache's keys and scales."""
    idx = s["idx"].reshape(-1, IDX_PAGE)
    return {"idx": idx[:, :PAGE * 128].view(torch.float8_e4m3fn), "idx_scale": idx[:, PAGE * 128:].view(torch.float32)}


def _plain_append(s):
    x = s["x"].float()
    rms = lambda v, w: ((v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5)) * w.float()).bfloat16()
    q = rms(x[:, :QL], s["g_q"]).float().reshape(-1, 16, 128)
    e = torch.ceil(torch.log2(q.abs().amax(-1).clamp(min=1e-10).double() / 448))
    qq = (q / torch.exp2(e).float()[..., None]).to(torch.float8_e4m3fn).reshape(-1, QL)
    b = (e + 127).int().reshape(-1, 4, 4)
    qsf = (b[..., 0] | (b[..., 1] << 8) | (b[..., 2] << 16) | (b[..., 3] << 24)).t().contiguous()
    cs = s["rope"][s["pos"].long()].float()
    turn = lambda v: torch.stack([v[:, 0::2] * cs[:, :32] - v[:, 1::2] * cs[:, 32:],
                                  v[:, 1::2] * cs[:, :32] + v[:, 0::2] * cs[:, 32:]], -1).reshape(-1, 64)
    kv = s["kv"]
    kv[s["slot"]] = _rows(rms(x[:, QL:QL + LAT], s["g_kv"]), turn(x[:, QL + LAT:QL + DIM]).bfloat16())
    out = {"q": qq, "qsf": qsf}
    if s["full"]:  # LayerNorm, rope on the first 64 dims, e4m3 with a power-of-two scale
        k = x[:, QL + DIM:]
        d = k - k.mean(-1, keepdim=True)
        k = d * torch.rsqrt(d.square().mean(-1, keepdim=True) + 1e-6) * s["ik_w"].float() + s["ik_b"].float()
        k = torch.cat([turn(k[:, :64]), k[:, 64:]], 1)
        sc = torch.exp2(torch.ceil(torch.log2(k.abs().amax(-1, keepdim=True).clamp(min=1e-4).double() / 448))).float()
        idx = s["idx"].reshape(-1, IDX_PAGE)
        page, row = s["slot"] // PAGE, s["slot"] % PAGE
        cols = torch.arange(128, device=DEV)
        idx[page[:, None], row[:, None] * 128 + cols] = (k / sc).to(torch.float8_e4m3fn).view(torch.uint8)
        idx[page[:, None], PAGE * 128 + row[:, None] * 4 + cols[:4]] = sc.view(torch.uint8).reshape(-1, 4)
        out |= _index(s)
    slots, ok = _slots(s)
    out["kvd"] = _lift(kv[slots[ok]]).bfloat16()
    return out


def _plain_attn(s):
    x, k, live, _, _ = _scores(s)
    p, lse = _softmax(x)
    full = torch.zeros(*live.shape, s["H"], s["top"], device=DEV)
    full[live] = p
    o = torch.bmm(full.reshape(s["nseq"], -1, s["top"]), k[..., :LAT])
    return {"out": o.reshape(*live.shape, s["H"], LAT)[live].bfloat16(), "lse": lse}


def _plain_picks(s):
    at = torch.arange(TOPK, device=DEV)
    ok = (at[None] < s["tlen"][:, None]) & (s["ind"] >= 0)
    slots = torch.where(ok, s["ind"], 0).long()
    k = _lift(s["kv"])[slots]
    x = torch.bmm(s["q"].float(), k.transpose(1, 2)) * SCALE
    p, lse = _softmax(torch.where(ok[:, None], x, -torch.inf))
    return {"out": torch.bmm(p, k[..., :LAT]).bfloat16(), "lse": lse}


def _plain_weights(s):
    x, _, live, slots, ok = _scores(s)
    w = torch.zeros(*live.shape, s["top"], device=DEV)
    lse = torch.where(torch.isinf(s["lse"]), torch.zeros_like(s["lse"]), s["lse"])
    w[live] = torch.exp(x - lse[..., None]).sum(1)
    acc = s["acc"].clone()
    acc[slots[ok]] += w.sum(1)[ok]
    return {"acc": acc}


def _plain_evict(s):
    slots, ok = _slots(s)
    b = (s["acc"] + 0.0)[slots].view(torch.int32).long()
    key = torch.where(b < 0, -2147483648 - b, b)  # ordered as the floats are
    pos, n = s["pos"][slots], s["lens"][:, None].long()
    held = (pos < s["sink"]) | (pos >= s["seen"][:, None] - s["recent"])
    key = torch.where(held, 1 << 40, key)
    key = torch.where(ok, key, -(1 << 40))
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    keep = torch.zeros_like(ok)
    new = n.clamp(max=s["budget"])
    at = torch.arange(s["top"], device=DEV)[None]
    keep.scatter_(1, order, at < new)
    hole, mover = ~keep & (at < new), keep & (at >= new)
    count = hole.sum(1)
    moves, k = s["moves"], torch.arange(s["budget"], device=DEV)[None]
    inside = k < count[:, None]
    moves[..., 0][inside] = slots[hole].int()
    moves[..., 1][inside] = slots[mover].int()
    s["n_moves"].copy_(count)
    s["new_lens"].copy_(new[:, 0])
    pair = moves[inside].long()
    s["kv"][pair[:, 0]] = s["kv"][pair[:, 1]]
    return {"moves": moves, "n_moves": s["n_moves"], "new_lens": s["new_lens"], "kv": s["kv"]}


# ------------------------------------------------------------------------------------------ a pass

def run(s):
    kind = s["kind"]
    if not own:
        return {"append": _plain_append, "attn": _plain_attn, "picks": _plain_picks, "weights": _plain_weights,
                "evict": _plain_evict}[kind](s)
    import glmkv
    T = s["T"]
    if kind == "append":
        a = (s["x"], s["x"].shape[1], s["g_q"], s["g_kv"], s["rope"], s["pos"], s["slot"], s["kv"])
        z = (s["qq"], s["qsf"].view(torch.uint8), T, T)
        if s["full"]:
            glmkv.mla_prep_full(*a, s["idx"], s["ik_w"], s["ik_b"], *z, kv_dtype="fp4")
        else:
            glmkv.mla_prep_shared(*a, *z, kv_dtype="fp4")
        glmkv.kv4_dequant(s["kv"], s["bt"], s["max_pages"], s["lens"], s["nseq"], s["kvd"])
        return {"q": s["qq"].view(torch.float8_e4m3fn), "qsf": s["qsf"], "kvd": s["kvd"],
                **(_index(s) if s["full"] else {})}
    if kind == "attn":
        glmkv.kv4_attn(s["q"], s["kv"], s["n_pages"], s["bt"], s["max_pages"], s["cu"], s["lens"], s["nseq"], s["H"],
                       SCALE, s["out"], s["lse"], s["ws"], WORKSPACE, T)
        return {"out": s["out"], "lse": s["lse"]}
    if kind == "picks":
        glmkv.kv4_attn_picks(s["q"], s["kv"], s["n_pages"], s["ind"], s["tlen"], s["H"], SCALE, s["out"], s["lse"],
                             s["ws"], WORKSPACE, T)
        return {"out": s["out"], "lse": s["lse"]}
    if kind == "weights":
        acc = s["acc"].clone()  # each pass adds to the same sums
        glmkv.kv4_weights(s["q"], s["lse"], s["kv"], s["n_pages"], s["bt"], s["max_pages"], s["cu"], s["lens"],
                          s["nseq"], s["H"], SCALE, acc, T)
        return {"acc": acc}
    glmkv.evict_plan(s["acc"], s["pos"], s["n_pages"], s["bt"], s["max_pages"], s["lens"], s["seen"], s["nseq"],
                     s["budget"], s["sink"], s["recent"], s["moves"], s["n_moves"], s["new_lens"])
    glmkv.evict_rows(s["moves"], s["n_moves"], s["nseq"], s["budget"], s["n_pages"], s["kv"], None, None, None,
                     kv_dtype="fp4")
    return {"moves": s["moves"], "n_moves": s["n_moves"], "new_lens": s["new_lens"], "kv": s["kv"]}


# ------------------------------------------------------------------------------------------ floors and 64 bits

def work(case):
    prefix, fresh = _shape(case)
    T, kind = sum(fresh), case["kind"]
    keys = sum(prefix) + T
    if kind == "append":
        x = 2 * (QL + DIM) + (256 if case["full"] else 0)
        return {"bytes": T * (x + 128 + 12 + QL + 16 + ROW + (132 if case["full"] else 0) + ROW + 2 * DIM),
                "flops": T * (4 * QL + 8 * LAT)}
    if kind == "evict":
        new = [min(p, case["budget"]) for p in prefix]
        # rows that move: with scores independent of the place, the dropped share of the kept range
        moves = sum(n * (p - n) // p for p, n in zip(prefix, new))
        return {"bytes": 8 * keys + moves * (8 + 2 * ROW) + 12 * len(new), "flops": 4 * keys}
    H = case["heads"]
    if kind == "picks":
        pairs = sum(min(TOPK, p + t + 1) for p, f in zip(prefix, fresh) for t in range(f))
        # a key picked by several rows needs reading once
        read = sum(min(p + f, sum(min(TOPK, p + t + 1) for t in range(f))) for p, f in zip(prefix, fresh))
        return {"bytes": read * ROW + pairs * 4 + T * H * (2 * DIM + 2 * LAT + 4), "flops": 2 * (DIM + LAT) * pairs * H}
    pairs = sum(max(0, p + t + 1) for p, f in zip(prefix, fresh) for t in range(f))
    if kind == "weights":
        return {"bytes": keys * (ROW + 8) + T * H * (2 * DIM + 4), "flops": 2 * DIM * pairs * H}
    return {"bytes": keys * ROW + T * H * (2 * DIM + 2 * LAT + 4), "flops": 2 * (DIM + LAT) * pairs * H}


def _decode64(rows):
    """Cache rows in 64 bits, from the bits of the formats."""
    n = torch.stack([rows[:, :256] % 16, rows[:, :256] // 16], -1).reshape(-1, LAT).long()
    e, m = (n // 2) % 4, (n % 2).double()
    v = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2((e - 1).double())) * (1 - 2 * (n // 8).double())
    s = rows[:, 256:288].long()
    se, sm = (s // 8) % 16, (s % 8).double()
    sc = torch.where(se == 0, sm / 8 * 2.0 ** -6, (1 + sm / 8) * torch.exp2((se - 7).double()))
    u = rows[:, 288:].long()
    pe = ((u[:, 0::2] + 256 * u[:, 1::2]) << 16).to(torch.int32).view(torch.float32).double()
    return (v.reshape(-1, 32, 16) * sc[..., None]).reshape(-1, LAT), pe


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "append":
        # its outputs are codes and their scales, which a sum next to a rounding border puts on either side of
        # it: they have no value in 64 bits to be near to
        return None
    if kind == "evict":
        return None  # whole numbers and moved bytes
    H, cu, lens, bt = s["H"], s["cu"].tolist(), s["lens"].tolist(), s["bt"].long()
    outs, lses = [], []
    acc = s["acc"].double().clone() if kind == "weights" else None
    for i in range(s["nseq"]):
        j = torch.arange(lens[i], device=DEV)
        slots = bt[i, j // PAGE] * PAGE + j % PAGE
        rows = range(cu[i], cu[i + 1])
        for r in rows:
            if kind == "picks":
                at = s["ind"][r, :int(s["tlen"][r])].long()
            else:
                at = slots[:max(0, lens[i] - len(rows) + (r - cu[i]) + 1)]
            c, pe = _decode64(s["kv"][at])
            q = s["q"][r].double()
            x = (q[:, :LAT] @ c.T + q[:, LAT:] @ pe.T) * SCALE
            if kind == "weights":
                acc[at] += torch.exp(x - s["lse"][r].double()[:, None]).sum(0)
                continue
            if not len(at):
                outs.append(torch.zeros(H, LAT, dtype=torch.float64, device=DEV))
                lses.append(torch.full((H,), -torch.inf, dtype=torch.float64, device=DEV))
                continue
            lse = torch.logsumexp(x, 1)
            outs.append(torch.exp(x - lse[:, None]) @ c)
            lses.append(lse)
    if kind == "weights":
        return {"acc": acc}
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}
