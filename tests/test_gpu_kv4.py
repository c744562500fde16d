"""The 4-bit latent cache on the GPU: append, lift, attention and weights against oracle/kv4.py in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _np(t):
    return t.float().cpu().numpy() if t.dtype == torch.bfloat16 else t.cpu().numpy()


# ------------------------------------------------------------------------------------------ append and lift

def _append(cuda, x, lda, T, slot, kv_dtype, row, n_pages, full, seed=5, offset=0):
    import glmkv
    from glmkv import workload as W

    rng = np.random.default_rng(seed)
    w = W.weights(rng)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    b = lambda a: t(a.view(np.int16)).view(torch.bfloat16)
    buf = torch.zeros(x.size + 8, dtype=torch.bfloat16, device=cuda)
    buf[offset:offset + x.size] = b(x.reshape(-1))
    xs = buf[offset:offset + x.size]
    kv = torch.full((n_pages * 64, row), 0xA5, dtype=torch.uint8, device=cuda)
    idx = torch.zeros(n_pages * 64 * 132, dtype=torch.uint8, device=cuda)
    qq, qsf = (torch.zeros(n, dtype=torch.uint8, device=cuda) for n in (T * 2048, 16 * T))
    pos = t(rng.integers(0, 500, T).astype(np.int32))
    a = (xs, lda, b(w.g_q), b(w.g_kv), b(W.rope_table(512)), pos, t(slot), kv)
    if full:
        glmkv.mla_prep_full(*a, idx, b(w.ik_w), b(w.ik_b), qq, qsf, T, T, kv_dtype=kv_dtype)
    else:
        glmkv.mla_prep_shared(*a, qq, qsf, T, T, kv_dtype=kv_dtype)
    torch.cuda.synchronize()
    assert glmkv.fault_flags() == 0
    return [_np(v) for v in (kv, idx, qq, qsf)]


@pytest.mark.parametrize("T,full,lda,offset", [(1, False, 2624, 0), (77, True, 2752, 0), (300, False, 2752, 0),
                                               (65, True, 2756, 4), (2500, True, 2752, 0)])
def test_append_is_the_packed_bf16_row(cuda, T, full, lda, offset):
    """The row is bit for bit the definition applied to the bf16 append's row, and all else is that append's."""
    from glmkv import workload as W
    from oracle import kv4

    rng = np.random.default_rng(T)
    xf = rng.standard_normal((T, lda)) * np.exp2(rng.integers(-6, 7, (T, 1)))
    xf[::7, 2048:2048 + 128] = 0                       # groups of zeros
    xf[3::11, 2048 + 16:2048 + 32] *= 1e-3             # scales near e4m3's smallest
    xf[5::13, 2048 + 32:2048 + 40] *= 1e4              # a group with one tall half
    if T > 2:
        xf[2, 2048:2560] = 0                           # a zero row
    x = W.bf16_bits(xf.astype(np.float32))
    n_pages = T // 64 + 3
    slot = rng.permutation(n_pages * 64)[:T].astype(np.int64)
    if T > 10:
        slot[4] = -1                                   # no cache slot
    kv4_, idx4, qq4, qsf4 = _append(cuda, x, lda, T, slot, "fp4", 416, n_pages, full, offset=offset)
    kvb, idxb, qqb, qsfb = _append(cuda, x, lda, T, slot, "bf16", 1152, n_pages, full, offset=offset)
    assert np.array_equal(idx4, idxb) and np.array_equal(qq4, qqb) and np.array_equal(qsf4, qsfb)
    live = slot[slot >= 0]
    bits = kvb[live].copy().view(np.uint16)
    want = np.full_like(kv4_, 0xA5)
    want[live] = kv4.pack(kv4.bf16_value(bits[:, :512]), bits[:, 512:])
    bad = np.argwhere(want != kv4_)
    assert len(bad) == 0, f"{len(bad)} bytes differ, first at {bad[:4].tolist()}"


@pytest.mark.parametrize("last", [1.0, float("inf"), float("nan")])
def test_append_over_the_formats_range(cuda, last):
    """Gains from 2^-16 to 2^14, 16 columns each: groups that become zeros, scales of fewer than four bits, scales that
    saturate; one infinite or NaN latent, and a row with an infinite input. The row is the packed bf16 row throughout."""
    import glmkv
    from glmkv import workload as W
    from oracle import kv4

    rng = np.random.default_rng(8)
    T, n_pages = 50, 1
    w = W.weights(rng)
    gains = np.repeat(np.exp2(np.arange(32) - 16.0), 16).astype(np.float32)
    gains[31 * 16:] = 1.0
    gains[511] = last
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    b = lambda a: t(a.view(np.int16)).view(torch.bfloat16)
    xf = rng.standard_normal((T, 2624)).astype(np.float32)
    xf[3, 2048 + 100] = np.inf                          # the norm's factor is 0, this latent 0 * inf
    x = W.bf16_bits(xf)
    got = {}
    for kv_dtype, row in (("fp4", 416), ("bf16", 1152)):
        kv = torch.full((n_pages * 64, row), 0xA5, dtype=torch.uint8, device=cuda)
        qq, qsf = (torch.zeros(n, dtype=torch.uint8, device=cuda) for n in (T * 2048, 16 * T))
        glmkv.mla_prep_shared(b(x), 2624, b(w.g_q), b(W.bf16_bits(gains)), b(W.rope_table(64)),
                              torch.zeros(T, dtype=torch.int32, device=cuda), torch.arange(T, device=cuda), kv, qq, qsf, T,
                              T, kv_dtype=kv_dtype)
        torch.cuda.synchronize()
        got[kv_dtype] = kv.cpu().numpy()[:T]
    assert glmkv.fault_flags() == 0
    rows, bits = got["fp4"], got["bf16"].copy().view(np.uint16)
    v = kv4.bf16_value(bits[:, :512])
    # a group with a NaN is NaN as a whole, by its scale; its codes say nothing
    nan = np.isnan(v).reshape(T, 32, 16).any(-1)
    assert nan[3].any() and nan[:, 31].all() == np.isnan(last)
    assert np.array_equal((rows[:, 256:288] & 0x7F) == 0x7F, nan)
    v[np.repeat(nan, 16, 1)] = 0
    rows[:, 256:288][nan], rows[:, :256][np.repeat(nan, 8, 1)] = 0, 0
    want = kv4.pack(v, bits[:, 512:])
    assert np.array_equal(rows, want)
    lat = kv4.lift(rows)[0]
    top = np.abs(v.reshape(T, 32, 16)).max(-1)
    assert not lat.reshape(T, 32, 16)[top < 6 * 2.0 ** -10].any() and (top < 6 * 2.0 ** -10).any()
    if np.isinf(last):
        rest = np.arange(T) != 3
        assert np.array_equal(lat[rest, 511], np.sign(v[rest, 511]) * 2688)


@pytest.mark.parametrize("lens", [[1], [63, 0, 64, 65, 1], [700, 1, 129, 4000], [0, 0]])
def test_lift_is_exact(cuda, lens):
    import glmkv
    from kv4_case import Kv4Case
    from oracle import kv4

    c = Kv4Case(lens, [0] * len(lens), 1, seed=len(lens))
    d = c.device(torch, cuda)
    kvd = torch.full((sum(lens) + 3, 576), 7.0, dtype=torch.bfloat16, device=cuda)
    glmkv.kv4_dequant(d["kv"], d["bt"], c.max_pages, d["lens"], c.nseq, kvd)
    torch.cuda.synchronize()
    assert glmkv.fault_flags() == 0
    rows = np.concatenate([c.kv[kv4.slots_of(c.bt, s, n)] for s, n in enumerate(lens)])
    want = np.concatenate(kv4.lift(rows), 1) if len(rows) else np.zeros((0, 576))
    assert np.array_equal(_np(kvd)[:sum(lens)].astype(np.float64), want)
    assert np.all(_np(kvd)[sum(lens):] == 7.0)


# ------------------------------------------------------------------------------------------ attention

CASES = [  # cached tokens, query tokens, heads
    ([1], [1], 1),
    ([5], [1], 64),
    ([128], [1], 64),
    ([129, 64, 1], [1, 1, 1], 16),
    ([0, 300, 0], [1, 1, 2], 8),               # sequences with nothing cached: empty rows
    ([2, 40], [5, 3], 24),                     # more query tokens than cached ones: empty rows first
    ([1000], [3], 40),                         # row tiles across query tokens
    ([700, 0, 130], [1, 0, 4], 128),           # a sequence without query tokens
    ([2000, 33, 4097], [1, 1, 1], 64),
    ([20000], [1], 128),                       # split over every CTA
    ([260, 250], [130, 250], 5),               # prompts, one of them from its first token
    ([70] * 200, [1] * 200, 64),               # more sequences than CTAs
]


@pytest.mark.parametrize("lens,qlens,heads", CASES)
def test_attention(cuda, lens, qlens, heads):
    import glmkv
    from kv4_case import Kv4Case

    c = Kv4Case(lens, qlens, heads, seed=heads)
    d = c.device(torch, cuda, pad=2)
    c.attn(d)
    torch.cuda.synchronize()
    assert glmkv.fault_flags() == 0
    out, lse = _np(d["out"]), _np(d["lse"])
    c.check_attn(out[:c.T], lse[:c.T])
    assert np.all(out[c.T:] == 7.0) and np.all(lse[c.T:] == 7.0)  # rows behind the last sequence


@pytest.mark.parametrize("q_std,scale", [(12.0, None), (1e-20, None), (1e20, 1e-20), (1.2, -0.06), (1.2, 0.0)])
def test_attention_of_sharp_flat_and_scaled_rows(cuda, q_std, scale):
    """Scores far apart (the reference is raised again and again), all alike, and q far from 1."""
    from kv4_case import Kv4Case

    c = Kv4Case([1500, 77], [2, 1], 64, seed=9, q_std=q_std)
    c.scale = c.scale if scale is None else scale
    d = c.device(torch, cuda)
    c.attn(d)
    c.check_attn(_np(d["out"]), _np(d["lse"]))


def _check_far(c, d):
    """Scores so large that their rounding in f32 is many powers of two: a row whose largest one leads by more than
    twice the scores' error and 40 more has that token's latents, which bf16 holds exactly, and its score for lse. A
    score's error: a sum of 576 products in f32, twice that with a truncating adder, and its factors' roundings. The
    tokens behind weigh 2^-57 each or less, and the output is off by its own rounding and the reciprocal's, together
    below 2^-8. lse is off by the score's error and two roundings."""
    from oracle import kv4

    out, lse = _np(d["out"]).astype(np.float64), _np(d["lse"]).astype(np.float64)
    assert np.all(np.isfinite(out)) and np.all(np.isfinite(lse))
    sure = 0
    for t in range(c.T):
        lat, pe = kv4.lift(c.kv[c.rows_of(t)])
        k = np.concatenate([lat, pe], 1)
        x = c.scale * (c.q[t] @ k.T)
        ds = (abs(c.scale) * (np.abs(c.q[t]) @ np.abs(k).T)).max(1) * 578 * 2.0 ** -23
        first, second = np.sort(x, 1)[:, -1], np.sort(x, 1)[:, -2]
        lead = first - second > 2 * ds + 40
        sure += lead.sum()
        want = lat[x.argmax(1)]
        assert np.all((np.abs(out[t] - want) <= np.abs(want) * 2.0 ** -8 + 2.0 ** -40)[lead])
        assert np.all((np.abs(lse[t] - first) <= ds + np.abs(first) * 2.0 ** -22)[lead])
    assert sure > 0.9 * c.T * c.heads


FAR = [(3e6, [200, 90], [2, 1]), (3e7, [200, 90], [2, 1]), (1e9, [1500, 77], [2, 1]), (-1e12, [1500, 77], [2, 1]),
       (1e30, [300, 129], [1, 1]), (1e9, [20000], [1])]


@pytest.mark.parametrize("scale,lens,qlens", FAR)
def test_attention_of_far_scores(cuda, scale, lens, qlens):
    """A reference past 2^28 is rounded by more than a weight's exponent has room for."""
    from kv4_case import Kv4Case

    c = Kv4Case(lens, qlens, 64, seed=13)
    c.scale = scale
    d = c.device(torch, cuda)
    c.attn(d)
    _check_far(c, d)


@pytest.mark.parametrize("scale", [1e9, 1e29])
@pytest.mark.parametrize("n", [100, 300, 20000])
def test_attention_of_scores_far_below_zero(cuda, scale, n):
    """Every score of a row below the reference that a row starts with, in a first tile and in later ones."""
    from kv4_case import Kv4Case, bf16
    from oracle import kv4

    c = Kv4Case([n], [1], 48, seed=14)
    lat, pe = bf16(np.abs(c.rng.standard_normal((n, 512)))), bf16(np.abs(c.rng.standard_normal((n, 64))))
    c.kv[kv4.slots_of(c.bt, 0, n)] = kv4.pack(lat[1], pe[0])
    c.q_bits, c.q = bf16(-np.abs(c.rng.standard_normal(c.q.shape)))
    c.scale = scale
    d = c.device(torch, cuda)
    c.attn(d)
    _check_far(c, d)


def test_attention_rising_scores(cuda):
    """Every tile's scores pass the last one's: the rows are rescaled a tile."""
    from kv4_case import Kv4Case, bf16
    from oracle import kv4

    c = Kv4Case([2000], [1], 32, seed=3)
    lat = np.ones((2000, 512)) * (1 + np.arange(2000)[:, None] / 200)
    c.kv[kv4.slots_of(c.bt, 0, 2000)] = kv4.pack(bf16(lat)[1], bf16(np.zeros((2000, 64)))[0])
    c.q_bits, c.q = bf16(np.abs(c.rng.standard_normal((1, 32, 576))))
    d = c.device(torch, cuda)
    c.attn(d)
    c.check_attn(_np(d["out"]), _np(d["lse"]))


def test_attention_keeps_nan_to_its_row(cuda):
    from kv4_case import Kv4Case

    c = Kv4Case([300], [2], 20, seed=4)
    clean = c.device(torch, cuda)
    c.attn(clean)
    d = c.device(torch, cuda)
    d["q"][1, 3, 7] = float("nan")
    c.attn(d)
    out, lse = _np(d["out"]), _np(d["lse"])
    assert np.all(np.isnan(out[1, 3])) and np.isnan(lse[1, 3])
    want, wlse = _np(clean["out"]), _np(clean["lse"])
    want[1, 3], wlse[1, 3] = np.nan, np.nan
    assert np.array_equal(out, want, equal_nan=True) and np.array_equal(lse, wlse, equal_nan=True)


@pytest.mark.parametrize("heads", [64, 16])
@pytest.mark.parametrize("at,byte", [(297, 256), (296, 287), (299, 288), (150, 270)])
def test_attention_keeps_a_nan_token_from_rows_before_it(cuda, heads, at, byte):
    """A cached token with a NaN scale, or a NaN key dim, makes NaN of the rows that see it and of no other."""
    import glmkv
    from kv4_case import Kv4Case
    from oracle import kv4

    c = Kv4Case([300], [6], heads, seed=7)
    d = c.device(torch, cuda)
    c.attn(d)
    want, wlse = _np(d["out"]), _np(d["lse"])
    row = kv4.slots_of(c.bt, 0, 300)[at]
    d["kv"][row, byte] = 0x7F if byte < 288 else 0xFF
    if byte >= 288:
        d["kv"][row, byte + 1] = 0x7F                  # bf16 0x7FFF
    c.attn(d)
    torch.cuda.synchronize()
    assert glmkv.fault_flags() == 0
    sees = 294 + np.arange(6) >= at
    want[sees], wlse[sees] = np.nan, np.nan
    assert np.array_equal(_np(d["out"]), want, equal_nan=True)
    assert np.array_equal(_np(d["lse"]), wlse, equal_nan=True)


@pytest.mark.parametrize("lens,heads,T", [([40], 64, 1), ([3000, 700], 40, 5), ([2500], 128, 9), ([2049, 1], 64, 300)])
def test_attention_over_picks(cuda, lens, heads, T):
    import glmkv
    from kv4_case import Kv4Case
    from oracle import kv4

    c = Kv4Case(lens, [T] + [0] * (len(lens) - 1), heads, seed=T)
    ind = np.full((T, 2048), -1, np.int32)
    tlen = np.zeros(T, np.int32)
    for t in range(T):
        s = t % len(lens)
        n = min(2048, int(c.rng.integers(0, lens[s] + 1)))
        if t == 1:
            n = 0                                                # a row with no picks at all
        at = np.sort(c.rng.choice(lens[s], n, replace=False))
        ind[t, :n], tlen[t] = kv4.slots_of(c.bt, s, lens[s])[at], n
        if n > 3:
            ind[t, 1] = -1                                       # skipped
            ind[t, 2] = ind[t, 0]                                # the same token twice counts twice
    d = c.device(torch, cuda)
    g = lambda a: torch.from_numpy(a).to(cuda)
    glmkv.kv4_attn_picks(d["q"], d["kv"], c.n_pages, g(ind), g(tlen), heads, c.scale, d["out"], d["lse"], d["ws"],
                         d["ws_bytes"], T)
    torch.cuda.synchronize()
    assert glmkv.fault_flags() == 0
    pick = lambda t: ind[t, :tlen[t]][ind[t, :tlen[t]] >= 0]
    c.check_attn(_np(d["out"]), _np(d["lse"]), rows_of=pick)


@pytest.mark.parametrize("lens,qlens,heads", CASES)
def test_weights(cuda, lens, qlens, heads):
    import glmkv
    from kv4_case import Kv4Case

    c = Kv4Case(lens, qlens, heads, seed=heads + 1)
    d = c.device(torch, cuda, pad=1)
    c.attn(d)
    start = torch.rand(c.n_pages * 64, device=cuda, generator=torch.Generator(cuda).manual_seed(1))
    acc = start.clone()
    c.weights(d, acc)
    again = start.clone()
    c.weights(d, again)
    torch.cuda.synchronize()
    assert glmkv.fault_flags() == 0
    assert torch.equal(acc, again)
    want, tol = c.want_weights(_np(d["lse"])[:c.T].astype(np.float64))
    got, s = _np(acc).astype(np.float64), _np(start).astype(np.float64)
    err = np.abs(got - (s + want))
    assert np.all(err <= tol + (s + want) * 2.0 ** -24), np.max(err)
    assert np.array_equal(got[want == 0], s[want == 0])
    rows = np.isfinite(_np(d["lse"])[:c.T]).sum()
    assert abs(want.sum() - rows) < 1e-3 * max(rows, 1)


def _short_sequences(kind):
    """Batches where every CTA walks several sequences, each of a few tiles or of one."""
    if kind == "one tile":
        return [70] * 1000, [1] * 1000
    rng = np.random.default_rng(600)
    lens = rng.choice([0, 1, 64, 128, 129, 256, 300, 384, 640], 600).tolist()
    return lens, rng.choice([0, 1, 1, 1, 2], 600).tolist()


@pytest.mark.parametrize("kind", ["one tile", "mixed"])
@pytest.mark.parametrize("heads", [8, 64])
def test_many_short_sequences_a_cta(cuda, kind, heads):
    """A sequence's first tile is prepared before it begins, from what the walk says of it: no warp may read that
    before the walk is there. Attention and weights, several times over."""
    import glmkv
    from kv4_case import Kv4Case

    c = Kv4Case(*_short_sequences(kind), heads, seed=heads)
    d = c.device(torch, cuda)
    c.attn(d)
    out, lse = d["out"].clone(), d["lse"].clone()
    accs = []
    for _ in range(6):
        c.attn(d)
        assert torch.equal(out, d["out"]) and torch.equal(lse, d["lse"])
        accs.append(torch.zeros(c.n_pages * 64, device=cuda))
        c.weights(d, accs[-1])
    torch.cuda.synchronize()
    assert glmkv.fault_flags() == 0
    c.check_attn(_np(out), _np(lse))
    want, tol = c.want_weights(_np(lse).astype(np.float64))
    err = np.abs(_np(accs[0]).astype(np.float64) - want)
    assert np.all(err <= tol + want * 2.0 ** -24), np.max(err)
    assert all(torch.equal(accs[0], a) for a in accs[1:])


# ------------------------------------------------------------------------------------------ as a program uses them

def test_bad_pages_and_picks_are_skipped_and_flagged(cuda):
    import glmkv
    from kv4_case import Kv4Case
    from oracle import kv4

    c = Kv4Case([500], [1], 16, seed=2)
    slots = kv4.slots_of(c.bt, 0, 500)
    for bad in (-3, c.n_pages, 1 << 30):
        d = c.device(torch, cuda)
        d["bt"][0, 2] = bad
        c.attn(d)
        torch.cuda.synchronize()
        assert glmkv.fault_flags() == 2
        c.check_attn(_np(d["out"]), _np(d["lse"]), rows_of=lambda t: np.delete(slots, np.arange(128, 192)))
        acc = torch.zeros(c.n_pages * 64, device=cuda)
        c.weights(d, acc)
        assert glmkv.fault_flags() == 2
        assert np.all(_np(acc)[slots[128:192]] == 0)
    d = c.device(torch, cuda)
    c.attn(d, block_table=d["bt"][:, :4].contiguous(), max_pages=4)  # the table ends before the sequence
    assert glmkv.fault_flags() == 2
    c.check_attn(_np(d["out"]), _np(d["lse"]), rows_of=lambda t: slots[:256])
    ind = torch.full((1, 2048), -1, dtype=torch.int32, device=cuda)
    ind[0, 0], ind[0, 1] = int(slots[7]), c.n_pages * 64
    d = c.device(torch, cuda)
    glmkv.kv4_attn_picks(d["q"], d["kv"], c.n_pages, ind, torch.full((1,), 9, dtype=torch.int32, device=cuda), 16,
                         c.scale, d["out"], d["lse"], d["ws"], d["ws_bytes"], 1)
    assert glmkv.fault_flags() == 4
    c.check_attn(_np(d["out"]), _np(d["lse"]), rows_of=lambda t: slots[7:8])


def test_streams_and_graphs(cuda):
    """Two calls at once on streams of their own, and a captured call replayed on new inputs."""
    from kv4_case import Kv4Case

    a, b = Kv4Case([3000, 100], [1, 2], 64, seed=1), Kv4Case([900] * 5, [1] * 5, 32, seed=2)
    da, db = a.device(torch, cuda), b.device(torch, cuda)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        a.attn(da, stream=s1)
        b.attn(db, stream=s2)
    torch.cuda.synchronize()
    a.check_attn(_np(da["out"]), _np(da["lse"]), what="first stream")
    b.check_attn(_np(db["out"]), _np(db["lse"]), what="second stream")
    acc = torch.zeros(a.n_pages * 64, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.attn(da)
        a.weights(da, acc)
    new = Kv4Case([3000, 100], [1, 2], 64, seed=8)
    dn = new.device(torch, cuda)
    for k in ("q", "kv", "bt"):
        da[k].copy_(dn[k])
    acc.zero_()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    new.check_attn(_np(da["out"]), _np(da["lse"]), what="replayed")
    want, tol = new.want_weights(_np(da["lse"]).astype(np.float64))
    assert np.all(np.abs(_np(acc) - 2 * want) <= 2 * tol + want * 2.0 ** -22)


def test_offsets_past_32_bits(cuda):
    """A pool of 4.5 GB with the sequences in its last pages: append, lift, attention, picks, weights and moves."""
    import glmkv
    from glmkv import workload as W
    from kv4_case import Kv4Case
    from oracle import kv4

    c = Kv4Case([500, 130], [2, 1], 16, seed=21)
    d = c.device(torch, cuda)
    n_pages = 170000
    shift = n_pages - c.n_pages
    kv = torch.empty(n_pages * 64, 416, dtype=torch.uint8, device=cuda)
    kv[shift * 64:] = d["kv"]
    d["kv"], c.n_pages = kv, n_pages
    d["bt"] = torch.where(d["bt"] >= 0, d["bt"] + shift, d["bt"])
    c.bt = np.where(c.bt >= 0, c.bt + shift, c.bt)
    small, c.kv = c.kv, None

    class Pool:  # the host's copy of the pool's used end, by slot
        def __getitem__(self, at):
            return small[np.asarray(at) - shift * 64]

    c.kv = Pool()
    c.attn(d)
    c.check_attn(_np(d["out"]), _np(d["lse"]))
    acc = torch.zeros(n_pages * 64, device=cuda)
    c.weights(d, acc)
    at = np.concatenate([kv4.slots_of(c.bt, s, int(n)) for s, n in enumerate(c.lens)])
    want, tol = c.want_weights(_np(d["lse"]).astype(np.float64))
    err = np.abs(_np(acc)[at].astype(np.float64) - want[at])
    assert np.all(err <= tol[at] + want[at] * 2.0 ** -24)
    ind = torch.full((c.T, 2048), -1, dtype=torch.int32, device=cuda)
    tlen = torch.full((c.T,), 130, dtype=torch.int32, device=cuda)
    picks = [kv4.slots_of(c.bt, s, 130) for s in (0, 0, 1)]
    for t in range(c.T):
        ind[t, :130] = torch.from_numpy(picks[t].astype(np.int32)).to(cuda)
    glmkv.kv4_attn_picks(d["q"], kv, n_pages, ind, tlen, 16, c.scale, d["out"], d["lse"], d["ws"], d["ws_bytes"], c.T)
    c.check_attn(_np(d["out"]), _np(d["lse"]), rows_of=lambda t: picks[t])
    kvd = torch.zeros(630, 576, dtype=torch.bfloat16, device=cuda)
    glmkv.kv4_dequant(kv, d["bt"], c.max_pages, d["lens"], c.nseq, kvd)
    assert np.array_equal(_np(kvd).astype(np.float64), np.concatenate(kv4.lift(c.kv[at]), 1))
    # the last slots of the pool: an append into them, and moves between them
    rng = np.random.default_rng(22)
    w = W.weights(rng)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    b = lambda a: t(a.view(np.int16)).view(torch.bfloat16)
    x = b(W.bf16_bits(rng.standard_normal((8, 2624)).astype(np.float32)))
    rows = {}
    for name, pool, first in (("far", kv, n_pages * 64 - 8), ("near", torch.zeros(64, 416, dtype=torch.uint8, device=cuda), 0)):
        qq, qsf = (torch.zeros(n, dtype=torch.uint8, device=cuda) for n in (8 * 2048, 16 * 8))
        glmkv.mla_prep_shared(x, 2624, b(w.g_q), b(w.g_kv), b(W.rope_table(64)), torch.arange(8, dtype=torch.int32, device=cuda),
                              torch.arange(first, first + 8, device=cuda), pool, qq, qsf, 8, 8, kv_dtype="fp4")
        rows[name] = _np(pool[first:first + 8])
    assert np.array_equal(rows["far"], rows["near"])
    moves = torch.tensor([[[n_pages * 64 - 1, n_pages * 64 - 8], [n_pages * 64 - 2, n_pages * 64 - 7]]], dtype=torch.int32,
                         device=cuda)
    glmkv.evict_rows(moves, torch.tensor([2], dtype=torch.int32, device=cuda), 1, 2, n_pages, kv, None, None, None)
    assert np.array_equal(_np(kv[-2:]), rows["near"][[1, 0]])
    assert glmkv.fault_flags() == 0


def test_same_bits_every_time(cuda):
    from kv4_case import Kv4Case

    c = Kv4Case([9000, 1300], [2, 1], 64, seed=6)
    d = c.device(torch, cuda)
    c.attn(d)
    out, lse = d["out"].clone(), d["lse"].clone()
    for _ in range(3):
        d["ws"].fill_(0xFF)
        c.attn(d)
        assert torch.equal(out, d["out"]) and torch.equal(lse, d["lse"])


def test_layer_group_with_four_bit_rows(cuda):
    """A stage's call with 4-bit rows: the caches hold the bf16 call's rows packed, the row plans are its own, and
    attention over the slots they leave agrees with 64 bits."""
    import glmkv
    from glmkv import stage, workload as W
    from kv4_case import Kv4Case, bf16
    from oracle import kv4

    rng = np.random.default_rng(31)
    call = W.make_call([130, 0, 2200], [3, 70, 5], rng, spare_pages=3)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    bf = lambda a: t(a.view(np.int16)).view(torch.bfloat16)
    meta = stage.CallMeta(t(call.cu), t(call.seq_lens), t(call.block_table), t(call.slot_mapping), call.nseq, call.T,
                          call.ctx)
    inputs, ind = {}, {}
    for l in range(4):
        w = W.weights(rng)
        full = l in stage.FULL
        inputs[l] = stage.LayerInputs(bf(W.activations(rng, call.T)), bf(w.g_q), bf(w.g_kv),
                                      bf(w.ik_w) if full else None, bf(w.ik_b) if full else None)
        if full:
            ind[l] = t(W.topk_indices(rng, call))
    n = call.n_pages * 64
    lat, pe = bf16(rng.standard_normal((n, 512))), bf16(rng.standard_normal((n, 64)))
    pools = {"fp4": kv4.pack(lat[1], pe[0]), "bf16": np.concatenate([lat[0], pe[0]], 1).view(np.uint8)}
    ipool = W.random_index_pages(rng, call.n_pages)
    groups, inds = {}, {}
    for dt, pool in pools.items():
        g = groups[dt] = stage.LayerGroup(0, 4, n_pages=call.n_pages, max_ctx=call.ctx, chunk=call.T, kv_dtype=dt,
                                          device=cuda)
        g.rope = bf(W.rope_table(int(call.seq_lens.max())))
        for l in g.kv:
            g.kv[l].copy_(t(pool.reshape(-1)))
        for l in g.idx:
            g.idx[l].copy_(t(ipool))
        inds[dt] = {l: v.clone() for l, v in ind.items()}
        seen = []
        g.run_call(meta, inputs, inds[dt], on_op=lambda op, l, before: seen.append((op, l)) if before else None)
        assert len(seen) == g.launches_per_call() and "kv_dequant" not in [op for op, _ in seen]
    torch.cuda.synchronize()
    a, b = groups["fp4"], groups["bf16"]
    for l in a.kv:
        rows, ref = _np(a.kv[l]).reshape(-1, 416), _np(b.kv[l]).reshape(-1, 1152).view(np.uint16)
        at = call.slot_mapping
        assert np.array_equal(rows[at], kv4.pack(kv4.bf16_value(ref[at, :512]), ref[at, 512:])), l
        kept = np.setdiff1d(np.arange(n), at)
        assert np.array_equal(rows[kept], pools["fp4"][kept]), l
    for l in a.idx:
        assert torch.equal(a.idx[l], b.idx[l]) and torch.equal(inds["fp4"][l], inds["bf16"][l])
    assert torch.equal(a.tlen, b.tlen)
    # layer 3 attends with the picks of layer 2
    heads = 64
    c = Kv4Case([int(x) for x in call.seq_lens], [int(x) for x in np.diff(call.cu)], heads, seed=2)
    d = c.device(torch, cuda)
    picks, tlen = _np(inds["fp4"][stage.picks_source(3)]), _np(a.tlen)
    glmkv.kv4_attn_picks(d["q"], a.kv[3], call.n_pages, inds["fp4"][stage.picks_source(3)], a.tlen, heads, c.scale,
                         d["out"], d["lse"], d["ws"], d["ws_bytes"], call.T)
    torch.cuda.synchronize()
    assert glmkv.fault_flags() == 0
    c.kv = _np(a.kv[3]).reshape(-1, 416)
    c.check_attn(_np(d["out"]), _np(d["lse"]),
                 rows_of=lambda i: picks[i, :tlen[i]][picks[i, :tlen[i]] >= 0].astype(np.int64))
