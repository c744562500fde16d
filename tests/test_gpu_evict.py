"""Eviction by accumulated weight, and the 4-bit operators run together as a serving loop runs them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _pool(lens, seed, spare=2):
    rng = np.random.default_rng(seed)
    pages = [(n + 63) // 64 for n in lens]
    n_pages, max_pages = sum(pages) + spare, max(1, *pages)
    perm = rng.permutation(n_pages).astype(np.int32)
    bt = np.full((len(lens), max_pages), -1, np.int32)
    at = 0
    for s, n in enumerate(pages):
        bt[s, :n] = perm[at:at + n]
        at += n
    return rng, n_pages, max_pages, bt


def _plan(cuda, acc, pos, n_pages, bt, lens, seen, budget, sink, recent, alias=False):
    import glmkv

    g = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    nseq = len(lens)
    moves = torch.full((nseq, budget, 2), -9, dtype=torch.int32, device=cuda)
    n_moves = torch.full((nseq,), -9, dtype=torch.int32, device=cuda)
    dl = g(np.array(lens, np.int32))
    new = dl if alias else torch.zeros_like(dl)
    glmkv.evict_plan(g(acc), g(pos), n_pages, g(bt), bt.shape[1], dl, g(np.array(seen, np.int32)), nseq, budget, sink,
                     recent, moves, n_moves, new)
    torch.cuda.synchronize()
    return moves.cpu().numpy(), n_moves.cpu().numpy(), new.cpu().numpy()


def _check_plan(acc, pos, bt, lens, seen, budget, sink, recent, moves, n_moves, new):
    from oracle import kv4

    for s, n in enumerate(lens):
        at = kv4.slots_of(bt, s, n)
        stay = kv4.keep(acc[at].astype(np.float64), pos[at], seen[s], budget, sink, recent)
        to, frm = kv4.moves(stay)
        assert new[s] == min(n, budget) and n_moves[s] == len(to), s
        assert np.array_equal(moves[s, :len(to), 0], at[to]) and np.array_equal(moves[s, :len(to), 1], at[frm]), s
        assert np.all(moves[s, len(to):] == -9), s  # entries past the moves are left as they were


WEIGHTS = {
    "spread": lambda r, n: np.exp(2 * r.standard_normal(n)),
    "ties": lambda r, n: r.integers(0, 4, n),
    "equal": lambda r, n: np.zeros(n),
    "signs": lambda r, n: np.where(r.random(n) < 0.3, -0.0, np.where(r.random(n) < 0.5, 0.0, r.standard_normal(n))),
    "odd": lambda r, n: r.choice([np.nan, np.inf, -np.inf, 1e-45, -1e-45, 3e38, 1.0, -np.nan], n),
}


@pytest.mark.parametrize("kind", WEIGHTS)
@pytest.mark.parametrize("lens,budget,sink,recent", [
    ([1], 1, 0, 0), ([2, 64, 65, 0, 1], 1, 1, 0), ([200, 128, 129, 5], 100, 4, 20), ([4000, 1], 0, 0, 0),
    ([5000, 64, 2049], 2049, 2048, 1), ([3001] * 30, 1500, 0, 1500), ([100000], 33333, 16, 1000)])
def test_plan(cuda, kind, lens, budget, sink, recent):
    import glmkv

    rng, n_pages, _, bt = _pool(lens, seed=len(lens))
    acc = WEIGHTS[kind](rng, n_pages * 64).astype(np.float32)
    pos = np.zeros(n_pages * 64, np.int32)
    seen = []
    from oracle import kv4
    for s, n in enumerate(lens):  # positions with gaps, out of order: tokens have been evicted before
        all_ = np.sort(rng.choice(3 * n + 5, n, replace=False))
        pos[kv4.slots_of(bt, s, n)] = rng.permutation(all_) if s % 2 else all_
        seen.append(int(all_[-1]) + 1 if n else 0)
    got = _plan(cuda, acc, pos, n_pages, bt, lens, seen, budget, sink, recent, alias=kind == "ties")
    assert glmkv.fault_flags() == 0
    _check_plan(acc, pos, bt, lens, seen, budget, sink, recent, *got)


def test_plan_of_a_very_long_sequence(cuda):
    """More tokens a CTA than its shared memory keeps keys for."""
    rng, n_pages, _, bt = _pool([900001], seed=1)
    acc = rng.random(n_pages * 64).astype(np.float32)
    pos = np.zeros(n_pages * 64, np.int32)
    from oracle import kv4
    pos[kv4.slots_of(bt, 0, 900001)] = np.arange(900001)
    got = _plan(cuda, acc, pos, n_pages, bt, [900001], [900001], 400000, 4, 64)
    _check_plan(acc, pos, bt, [900001], [900001], 400000, 4, 64, *got)


@pytest.mark.parametrize("kv_dtype,row", [("fp4", 416), ("fp8", 656), ("bf16", 1152)])
def test_rows_move(cuda, kv_dtype, row):
    import glmkv

    lens, budget = [300, 7, 1000, 64], 130
    rng, n_pages, _, bt = _pool(lens, seed=row)
    n = n_pages * 64
    acc, pos = rng.random(n).astype(np.float32), np.arange(n, dtype=np.int32)
    moves, n_moves, _ = _plan(cuda, acc, pos, n_pages, bt, lens, [10 ** 6] * 4, budget, 0, 0)
    g = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    kv, idx = rng.integers(0, 256, (n, row), dtype=np.uint8), rng.integers(0, 256, (n_pages, 8448), dtype=np.uint8)
    d = [g(a) for a in (kv, idx, acc, pos)]
    glmkv.evict_rows(g(moves), g(n_moves), 4, budget, n_pages, *d, kv_dtype=kv_dtype)
    torch.cuda.synchronize()
    assert glmkv.fault_flags() == 0
    keys, sc = idx[:, :8192].reshape(n, 128).copy(), idx[:, 8192:].reshape(n, 4).copy()
    kw, aw, pw = kv.copy(), acc.copy(), pos.copy()
    for s in range(4):
        to, frm = moves[s, :n_moves[s]].T
        for a in (kw, aw, pw, keys, sc):
            a[to] = a[frm]
    iw = np.concatenate([keys.reshape(n_pages, 8192), sc.reshape(n_pages, 256)], 1)
    for name, got, want in zip(("kv", "idx", "acc", "pos"), d, (kw, iw, aw, pw)):
        assert np.array_equal(got.cpu().numpy(), want), name
    # only what is named moves
    only = g(acc)
    glmkv.evict_rows(g(moves), g(n_moves), 4, budget, n_pages, None, None, only, None, kv_dtype=kv_dtype)
    assert np.array_equal(only.cpu().numpy(), aw)


def test_bad_slots_are_skipped_and_flagged(cuda):
    import glmkv

    lens = [500]
    rng, n_pages, _, bt = _pool(lens, seed=3)
    acc, pos = rng.random(n_pages * 64).astype(np.float32) + 1, np.full(n_pages * 64, 50, np.int32)
    bt[0, 1] = n_pages
    moves, n_moves, new = _plan(cuda, acc, pos, n_pages, bt, lens, [1000], 480, 0, 0)
    assert glmkv.fault_flags() == 2 and new[0] == 480
    kv = torch.zeros(n_pages * 64, 416, dtype=torch.uint8, device=cuda)
    g = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    glmkv.evict_rows(g(moves), g(n_moves), 1, 480, n_pages, kv, None, None, None)
    assert glmkv.fault_flags() == 2  # the holes in the missing page


def test_a_serving_loop(cuda):
    """Append, attention, weights, eviction, and attention over what is left: two rounds, against 64 bits on
    the rows the cache then holds."""
    import glmkv
    from glmkv import workload as W
    from kv4_case import bf16
    from oracle import kv4

    rng = np.random.default_rng(11)
    H, budget, sink, recent, nseq, max_pages, n_pages = 24, 150, 4, 32, 3, 4, 14
    w = W.weights(rng)
    g = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    b = lambda a: g(a.view(np.int16)).view(torch.bfloat16)
    bt = rng.permutation(n_pages)[:nseq * max_pages].reshape(nseq, max_pages).astype(np.int32)
    kv = torch.full((n_pages * 64, 416), 0x7F, dtype=torch.uint8, device=cuda)
    acc = torch.zeros(n_pages * 64, device=cuda)
    pos = torch.zeros(n_pages * 64, dtype=torch.int32, device=cuda)
    rope, dbt = b(W.rope_table(2048)), g(bt)
    n_ws = glmkv.kv4_workspace_bytes()
    ws = torch.empty(n_ws, dtype=torch.uint8, device=cuda)
    moves = torch.zeros(nseq, budget, 2, dtype=torch.int32, device=cuda)
    n_moves = torch.zeros(nseq, dtype=torch.int32, device=cuda)
    lens, seen = np.zeros(nseq, np.int32), np.zeros(nseq, np.int32)
    for fresh in ([200, 97, 3], [50, 80, 100], [1, 1, 1]):
        fresh = np.array(fresh, np.int32)
        T = int(fresh.sum())
        seq = np.repeat(np.arange(nseq), fresh)
        rel = np.concatenate([np.arange(f) for f in fresh])
        index, place = lens[seq] + rel, (seen[seq] + rel).astype(np.int32)
        slot = bt[seq, index // 64].astype(np.int64) * 64 + index % 64
        lens, seen = lens + fresh, seen + fresh
        x = W.activations(rng, T)
        qq, qsf = (torch.zeros(n, dtype=torch.uint8, device=cuda) for n in (T * 2048, 16 * T))
        glmkv.mla_prep_shared(b(x), x.shape[1], b(w.g_q), b(w.g_kv), rope, g(place), g(slot), kv, qq, qsf, T, T,
                              kv_dtype="fp4")
        pos[g(slot)] = g(place)
        acc[g(slot)] = 0
        cu, dl = g(np.concatenate([[0], np.cumsum(fresh)]).astype(np.int64)), g(lens)
        qb, q = bf16(rng.standard_normal((T, H, 576)))
        out = torch.zeros(T, H, 512, dtype=torch.bfloat16, device=cuda)
        lse = torch.zeros(T, H, device=cuda)
        glmkv.kv4_attn(b(qb), kv, n_pages, dbt, max_pages, cu, dl, nseq, H, 0.0625, out, lse, ws, n_ws, T)
        glmkv.kv4_weights(b(qb), lse, kv, n_pages, dbt, max_pages, cu, dl, nseq, H, 0.0625, acc, T)
        torch.cuda.synchronize()
        rows, o, ls = kv.cpu().numpy(), out.float().cpu().numpy(), lse.cpu().numpy()
        for t in range(T):
            s = seq[t]
            at = kv4.slots_of(bt, s, int(index[t]) + 1)
            want, wl, _, mag, smag, cmag = kv4.attend(q[t], rows[at], 0.0625)
            ds = smag[:, None] * 576 * 2.0 ** -23
            assert np.all(np.abs(o[t] - want) <= np.abs(want) * 2.0 ** -8 + mag * (2.0 ** -10 + 2 * ds) + cmag * 2.0 ** -32)
            assert np.all(np.abs(ls[t] - wl) <= ds[:, 0] + 2.0 ** -17)
        a, p = acc.cpu().numpy(), pos.cpu().numpy()
        glmkv.evict_plan(acc, pos, n_pages, dbt, max_pages, dl, g(seen), nseq, budget, sink, recent, moves, n_moves, dl)
        glmkv.evict_rows(moves, n_moves, nseq, budget, n_pages, kv, None, acc, pos)
        torch.cuda.synchronize()
        after = kv.cpu().numpy()
        for s in range(nseq):
            at = kv4.slots_of(bt, s, int(lens[s]))
            stay = kv4.keep(a[at].astype(np.float64), p[at], seen[s], budget, sink, recent)
            left = at[:int(stay.sum())]
            assert sorted(p[at][stay]) == sorted(pos.cpu().numpy()[left])
            have = {int(v): i for i, v in enumerate(p[at])}
            for j in left:
                assert np.array_equal(after[j], rows[at[have[int(pos[j])]]])
            lens[s] = stay.sum()
        assert np.array_equal(dl.cpu().numpy(), lens)
    assert glmkv.fault_flags() == 0


@pytest.mark.parametrize("nseq", [1, 3, 257, 700])
def test_plan_takes_positions_from_what_was_seen(cuda, nseq):
    import glmkv

    rng = np.random.default_rng(nseq)
    fresh = rng.integers(0, 6, nseq)
    fresh[-1] += 1
    lens = fresh + rng.integers(0, 200, nseq)
    seen = lens + rng.integers(0, 1000, nseq)
    cu = np.concatenate([[0], np.cumsum(fresh)])
    T = int(cu[-1])
    g = lambda a, dt=np.int32: torch.from_numpy(np.asarray(a).astype(dt)).to(cuda)
    outs = []
    for kw in ({}, {"seen": g(seen)}, {"seen": g(lens)}):
        o = [torch.full((T,), -7, dtype=torch.int32, device=cuda) for _ in range(6)]
        glmkv.plan(g(cu, np.int64), g(lens), nseq, *o, T, **kw)
        outs.append([v.cpu().numpy() for v in o])
    seq = np.repeat(np.arange(nseq), fresh)
    behind = cu[seq + 1] - np.arange(T)  # a row's distance from its sequence's end
    assert np.array_equal(outs[0][0], lens[seq] - behind) and np.array_equal(outs[1][0], seen[seq] - behind)
    for a, b in zip(outs[0][1:], outs[1][1:]):
        assert np.array_equal(a, b)
    for a, b in zip(outs[0], outs[2]):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("kv_dtype", ["fp4", "fp8", "bf16"])
def test_a_stage_goes_on_after_an_eviction(cuda, kv_dtype):
    """Two calls of a stage, its sequences cut between them, beside a stage whose are not: the second call's rows and
    indexer keys are the same bytes in both, whatever the sequences still hold."""
    import glmkv
    from glmkv import stage, workload as W
    from oracle import kv4

    rng = np.random.default_rng(17)
    nseq, max_pages, n_pages, budget, sink, recent = 3, 7, 23, 150, 4, 32
    row = {"fp4": 416, "fp8": 656, "bf16": 1152}[kv_dtype]
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    bf = lambda a: t(a.view(np.int16)).view(torch.bfloat16)
    bt = rng.permutation(n_pages)[:nseq * max_pages].reshape(nseq, max_pages).astype(np.int32)
    rope = bf(W.rope_table(1024))
    weights = {l: W.weights(rng) for l in range(4)}
    groups = {}
    for name in ("cut", "whole"):
        g = groups[name] = stage.LayerGroup(0, 4, n_pages=n_pages, max_ctx=nseq * max_pages * 64, chunk=512,
                                            kv_dtype=kv_dtype, device=cuda)
        g.rope = rope
        for v in [*g.kv.values(), *g.idx.values()]:
            v.zero_()
    lens = {name: np.zeros(nseq, np.int32) for name in groups}
    seen = np.zeros(nseq, np.int32)
    acc = t(rng.random(n_pages * 64).astype(np.float32))
    pos = torch.zeros(n_pages * 64, dtype=torch.int32, device=cuda)
    new = {}
    for step, fresh in enumerate([[300, 100, 64], [3, 90, 1]]):
        fresh = np.array(fresh, np.int32)
        T = int(fresh.sum())
        seq, rel = np.repeat(np.arange(nseq), fresh), np.concatenate([np.arange(f) for f in fresh])
        cu = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int64)
        x = {l: bf(W.activations(rng, T)) for l in range(4)}
        seen = seen + fresh
        for name, g in groups.items():
            at = lens[name][seq] + rel
            slot = bt[seq, at // 64].astype(np.int64) * 64 + at % 64
            lens[name] = lens[name] + fresh
            inputs = {l: stage.LayerInputs(x[l], bf(w.g_q), bf(w.g_kv), *((bf(w.ik_w), bf(w.ik_b)) if l in stage.FULL
                                                                         else ())) for l, w in weights.items()}
            ind = {l: torch.arange(2048, dtype=torch.int32, device=cuda).repeat(T, 1) for l in range(3)}
            meta = stage.CallMeta(t(cu), t(lens[name]), t(bt), t(slot), nseq, T, int(lens[name].sum()),
                                  seen=t(seen) if name == "cut" else None)
            g.run_call(meta, inputs, ind)
            torch.cuda.synchronize()
            new[name] = slot
            assert np.array_equal(g.pos[:T].cpu().numpy(), (seen[seq] - fresh[seq]) + rel)
            if name == "cut":
                pos[t(slot)] = g.pos[:T]
        rows = {n: {l: g.kv[l].cpu().numpy().reshape(-1, row) for l in g.kv} for n, g in groups.items()}
        keys = {n: {l: g.idx[l].cpu().numpy().reshape(n_pages, 8448) for l in g.idx} for n, g in groups.items()}
        key = lambda pool, s: (pool[s // 64, :8192].reshape(len(s), 64, 128)[np.arange(len(s)), s % 64],
                               pool[s // 64, 8192:].reshape(len(s), 64, 4)[np.arange(len(s)), s % 64])
        for l in range(4):
            assert np.array_equal(rows["cut"][l][new["cut"]], rows["whole"][l][new["whole"]]), (step, l)
        for l in range(3):
            for a, b in zip(key(keys["cut"][l], new["cut"]), key(keys["whole"][l], new["whole"])):
                assert np.array_equal(a, b), (step, l)
        if step == 0:
            g = groups["cut"]
            dl = t(lens["cut"])
            moves = torch.zeros(nseq, budget, 2, dtype=torch.int32, device=cuda)
            n_moves = torch.zeros(nseq, dtype=torch.int32, device=cuda)
            glmkv.evict_plan(acc, pos, n_pages, t(bt), max_pages, dl, t(seen), nseq, budget, sink, recent, moves, n_moves,
                             dl)
            for l in g.kv:
                glmkv.evict_rows(moves, n_moves, nseq, budget, n_pages, g.kv[l], g.idx.get(l), None, None,
                                 kv_dtype=kv_dtype)
            glmkv.evict_rows(moves, n_moves, nseq, budget, n_pages, None, None, acc, pos)
            torch.cuda.synchronize()
            lens["cut"] = dl.cpu().numpy()
            assert lens["cut"].tolist() == [150, 100, 64]
    # every survivor is the row of its position in the stage that lost none
    where = pos.cpu().numpy()
    for s in range(nseq):
        at = kv4.slots_of(bt, s, int(lens["cut"][s]))
        src = kv4.slots_of(bt, s, int(lens["whole"][s]))[where[at]]
        for l in range(4):
            assert np.array_equal(rows["cut"][l][at], rows["whole"][l][src])
    assert glmkv.fault_flags() == 0


def test_a_captured_step(cuda):
    """A whole step in one graph (plan, append, attention, weights, eviction), replayed from a fresh state: what the
    same calls outside a graph leave."""
    import glmkv
    from glmkv import workload as W
    from kv4_case import bf16

    rng = np.random.default_rng(23)
    H, nseq, max_pages, n_pages, budget, sink, recent = 16, 20, 3, 64, 70, 4, 16
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    b = lambda a: t(a.view(np.int16)).view(torch.bfloat16)
    lens = rng.integers(1, 160, nseq).astype(np.int32)
    fresh = np.minimum(lens, rng.integers(1, 4, nseq)).astype(np.int32)
    T = int(fresh.sum())
    bt = rng.permutation(n_pages)[:nseq * max_pages].reshape(nseq, max_pages).astype(np.int32)
    seq, rel = np.repeat(np.arange(nseq), fresh), np.concatenate([np.arange(f) for f in fresh])
    at = (lens - fresh)[seq] + rel
    slot = t(bt[seq, at // 64].astype(np.int64) * 64 + at % 64)
    w, x = W.weights(rng), b(W.activations(rng, T))
    g_q, g_kv, rope, dbt = b(w.g_q), b(w.g_kv), b(W.rope_table(4096)), t(bt)
    cu = t(np.concatenate([[0], np.cumsum(fresh)]).astype(np.int64))
    q = b(bf16(rng.standard_normal((T, H, 576)))[0])
    pos0 = np.zeros(n_pages * 64, np.int32)
    for s in range(nseq):
        j = np.arange(lens[s])
        pos0[bt[s, j // 64] * 64 + j % 64] = 10 * j
    start = {"kv": torch.randint(0, 120, (n_pages * 64, 416), dtype=torch.uint8, device=cuda), "pos": t(pos0),
             "acc": torch.rand(n_pages * 64, device=cuda), "lens": t(lens), "seen": t(10 * lens)}
    start["kv"][:, 256:288] = 0x38                     # scales of 1
    start["kv"][:, 288:] = 0
    d = {k: v.clone() for k, v in start.items()}
    o = {k: torch.zeros(T, dtype=torch.int32, device=cuda) for k in ("p", "ks", "ke", "klen", "row_seq", "zero")}
    qq, qsf = (torch.zeros(n, dtype=torch.uint8, device=cuda) for n in (T * 2048, 16 * T))
    out, lse = torch.zeros(T, H, 512, dtype=torch.bfloat16, device=cuda), torch.zeros(T, H, device=cuda)
    n_ws = glmkv.kv4_workspace_bytes()
    ws = torch.empty(n_ws, dtype=torch.uint8, device=cuda)
    moves, n_moves = (torch.zeros(n, dtype=torch.int32, device=cuda) for n in ((nseq, budget, 2), (nseq,)))

    def step():
        glmkv.plan(cu, d["lens"], nseq, *o.values(), T, seen=d["seen"])
        glmkv.mla_prep_shared(x, x.shape[1], g_q, g_kv, rope, o["p"], slot, d["kv"], qq, qsf, T, T, kv_dtype="fp4")
        d["pos"][slot] = o["p"]
        glmkv.kv4_attn(q, d["kv"], n_pages, dbt, max_pages, cu, d["lens"], nseq, H, 0.0625, out, lse, ws, n_ws, T)
        glmkv.kv4_weights(q, lse, d["kv"], n_pages, dbt, max_pages, cu, d["lens"], nseq, H, 0.0625, d["acc"], T)
        glmkv.evict_plan(d["acc"], d["pos"], n_pages, dbt, max_pages, d["lens"], d["seen"], nseq, budget, sink, recent, moves,
                         n_moves, d["lens"])
        glmkv.evict_rows(moves, n_moves, nseq, budget, n_pages, d["kv"], None, d["acc"], d["pos"])

    def results():
        torch.cuda.synchronize()
        return [v.clone() for v in (*d.values(), *o.values(), out, lse, n_moves)]

    step()
    want = results()
    assert int(n_moves.sum()) > 0 and int(want[3].max()) == budget
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        for k, v in start.items():
            d[k].copy_(v)
        out.zero_(), lse.zero_()
        graph.replay()
        for a, e in zip(results(), want):
            assert torch.equal(a, e)
    assert glmkv.fault_flags() == 0
