"""The 4-bit cache's operators without a GPU: the definition's own properties, and what the launchers refuse
on the host before any CUDA call."""
import numpy as np
import pytest

from oracle import kv4


def test_codes_round_to_nearest_even():
    v = np.zeros((1, 512))
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    v[0, :7], v[0, 7:14] = mids, [-m for m in mids]
    v[0, 15] = 6.0                               # amax 6: the scale is 1
    rows = kv4.pack(v, np.zeros((1, 64)))
    lat, pe = kv4.lift(rows)
    assert lat[0, :7].tolist() == [0, 1, 1, 2, 2, 4, 4] and lat[0, 7:14].tolist() == [0, -1, -1, -2, -2, -4, -4]
    assert lat[0, 15] == 6 and not lat[0, 16:].any() and not pe.any()


def test_lifted_values_fit_f16_and_bf16():
    x = np.outer(kv4.CODES, kv4.E4M3[:127]).reshape(-1)
    assert np.array_equal(x.astype(np.float16).astype(np.float64), x)
    b = x.astype(np.float32).view(np.uint32)
    assert not (b & 0xFFFF).any()


def test_scales_at_the_ends():
    assert kv4.E4M3[kv4.scales(np.array([0.0, 6 * 2.0 ** -11, 6 * 2.0 ** -9, 6.0, 2688.0, 1e30]))].tolist() == \
        [0, 0, 2.0 ** -9, 1, 448, 448]


@pytest.mark.parametrize("n,budget", [(1, 1), (10, 3), (100, 64), (100, 0), (5, 9)])
def test_moves_close_the_gaps(n, budget):
    rng = np.random.default_rng(n)
    acc = rng.integers(0, 3, n).astype(np.float64)
    stay = kv4.keep(acc, np.arange(n), n, budget, min(1, budget), min(1, budget))
    to, frm = kv4.moves(stay)
    kept = np.arange(n)
    kept[to] = frm
    assert sorted(kept[:stay.sum()]) == sorted(np.flatnonzero(stay)) and len(to) == len(frm)


def test_ties_go_to_the_lowest_index_and_nan_leaves_first():
    acc = np.array([1, np.nan, 2, 1, 1, -np.inf, 0.0, -0.0])
    assert np.flatnonzero(kv4.keep(acc, np.arange(8) + 5, 99, 3, 0, 0)).tolist() == [0, 2, 3]
    assert np.flatnonzero(kv4.keep(acc, np.arange(8) + 5, 99, 5, 0, 0)).tolist() == [0, 2, 3, 4, 6]
    assert np.flatnonzero(kv4.keep(acc, np.arange(8) + 5, 99, 7, 0, 0)).tolist() == [0, 2, 3, 4, 5, 6, 7]
    assert np.flatnonzero(kv4.keep(acc, np.arange(8), 8, 2, 0, 1)).tolist() == [2, 7]


A = 0x10000  # an aligned, never dereferenced address: every call below returns before any CUDA call
INF, NAN = float("inf"), float("nan")
CALLS = {  # launcher: a call that passes the host checks, and what changing an argument gives
    "glmkv_mla_prep_fp4": ([A, 2752, A, A, A, A, A, A, A, A, A, A, A, 64, 64, None],
                           {"ARG": [(1, 2740), (0, None), (9, None), (13, 32), (14, -1)],
                            "ALIGN": [(1, 2754), (0, A + 2), (7, A + 2)], "OK": [(14, 0)]}),
    "glmkv_kv4_dequant": ([A, A, 16, A, 2, A, None],
                          {"ARG": [(0, None), (1, None), (3, None), (5, None), (2, -1), (4, -1)],
                           "ALIGN": [(0, A + 8), (5, A + 8)], "OK": [(4, 0)]}),
    "glmkv_kv4_workspace_bytes": ([A], {"ARG": [(0, None)]}),
    # q, kv, n_pages, block_table, max_pages, cu, seq_lens, nseq, heads, scale, out, lse, ws, ws_bytes, T, stream
    "glmkv_kv4_attn": ([A, A, 9, A, 4, A, A, 2, 64, 0.06, A, A, A, 1 << 40, 8, None],
                       {"ARG": [(i, None) for i in (0, 1, 3, 5, 6, 10, 11, 12)] +
                               [(2, 0), (2, 1 << 26), (4, 0), (7, -1), (8, 0), (8, 1025), (9, INF), (9, NAN), (14, -1)],
                        "ALIGN": [(0, A + 8), (1, A + 8), (3, A + 2), (5, A + 4), (6, A + 2), (10, A + 8), (11, A + 2),
                                  (12, A + 8)], "OK": [(7, 0), (14, 0)]}),
    # q, kv, n_pages, ind, tlen, heads, scale, out, lse, ws, ws_bytes, T, stream
    "glmkv_kv4_attn_picks": ([A, A, 9, A, A, 64, 0.06, A, A, A, 1 << 40, 8, None],
                             {"ARG": [(i, None) for i in (0, 1, 3, 4, 7, 8, 9)] +
                                     [(2, 0), (5, 0), (5, 1025), (6, NAN), (11, -1)],
                              "ALIGN": [(0, A + 8), (1, A + 8), (3, A + 2), (4, A + 2), (7, A + 8), (8, A + 2), (9, A + 8)],
                              "OK": [(11, 0)]}),
    # q, lse, kv, n_pages, block_table, max_pages, cu, seq_lens, nseq, heads, scale, acc, T, stream
    "glmkv_kv4_weights": ([A, A, A, 9, A, 4, A, A, 2, 64, 0.06, A, 8, None],
                          {"ARG": [(i, None) for i in (0, 1, 2, 4, 6, 7, 11)] +
                                  [(3, 0), (5, 0), (8, -1), (9, 0), (10, -INF), (12, -1)],
                           "ALIGN": [(0, A + 8), (1, A + 2), (2, A + 8), (6, A + 4), (7, A + 2), (11, A + 2)],
                           "OK": [(8, 0), (12, 0)]}),
    # acc, pos, n_pages, block_table, max_pages, seq_lens, seen, nseq, budget, sink, recent, moves, n_moves, new_lens
    "glmkv_evict_plan": ([A, A, 9, A, 4, A, A, 2, 100, 4, 32, A, A, A, None],
                         {"ARG": [(i, None) for i in (0, 1, 3, 5, 6, 11, 12, 13)] +
                                 [(2, 0), (4, 0), (4, 1 << 26), (7, -1), (8, -1), (8, 35), (9, -1), (10, -1),
                                  (10, 2147483647)],
                          "ALIGN": [(0, A + 2), (1, A + 2), (3, A + 2), (5, A + 2), (6, A + 2), (11, A + 4), (12, A + 2),
                                    (13, A + 2)], "OK": [(7, 0)]}),
    # moves, n_moves, nseq, budget, n_pages, kv, row_bytes, idx, acc, pos
    "glmkv_evict_rows": ([A, A, 2, 100, 9, A, 416, A, A, A, None],
                         {"ARG": [(0, None), (1, None), (2, -1), (2, 65536), (3, -1), (4, 0), (6, 400)],
                          "ALIGN": [(0, A + 4), (1, A + 2), (5, A + 8), (7, A + 8), (8, A + 2), (9, A + 2)],
                          "OK": [(2, 0), (3, 0)]}),
}


@pytest.mark.parametrize("name", CALLS)
def test_host_side_argument_checks(built_lib, name):
    import torch

    import glmkv
    from glmkv import _lib

    fn = getattr(glmkv.lib(), name)
    good, changes = CALLS[name]
    want = {"ARG": _lib.ERR_ARG, "ALIGN": _lib.ERR_ALIGN, "OK": _lib.OK}
    for kind, at in changes.items():
        for i, v in at:
            args = list(good)
            args[i] = v
            assert fn(*args) == want[kind], (i, v)
    if not torch.cuda.is_available():  # the addresses are not real: only where the device query ends the call
        assert fn(*good) == _lib.ERR_DEVICE


def test_python_refusals(built_lib):
    import torch

    import glmkv

    t = torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ValueError, match="device memory"):
        glmkv.kv4_dequant(A, t, 1, A, 1, A, stream=0)
    with pytest.raises(TypeError, match="expected a CUDA tensor"):
        glmkv.evict_plan([1.0], A, 1, A, 1, A, A, 1, 1, 0, 0, A, A, A, stream=0)
    with pytest.raises(ValueError, match="kv_dtype"):
        glmkv.evict_rows(A, A, 1, 1, 1, A, None, None, None, kv_dtype="int8", stream=0)
    with pytest.raises(glmkv.GlmKvError, match="invalid argument"):
        glmkv.kv4_attn(A, A, 0, A, 1, A, A, 1, 64, 1.0, A, A, A, 0, 1, stream=0)


@pytest.mark.parametrize("kv_dtype", ["FP4", "nvfp4", "int4", "bfloat16", "", None])
def test_an_unknown_row_format_is_refused(built_lib, kv_dtype):
    """The append writes by it: bf16 rows in a 4-bit cache would end 2.8 times as far."""
    import glmkv
    from glmkv import workload as W

    with pytest.raises(ValueError, match="kv_dtype"):
        glmkv.mla_prep_full(A, 2752, A, A, A, A, A, A, A, A, A, A, A, 64, 64, kv_dtype=kv_dtype, stream=0)
    with pytest.raises(ValueError, match="kv_dtype"):
        glmkv.mla_prep_shared(A, 2752, A, A, A, A, A, A, A, A, 64, 64, kv_dtype=kv_dtype, stream=0)
    with pytest.raises(ValueError, match="kv_dtype"):
        W.random_latent_pages(np.random.default_rng(0), 1, kv_dtype)


class _OnDevice1:
    """Stands in for torch.Tensor in the bindings' eyes: a contiguous tensor of cuda:1."""

    def __init__(self, dtype):
        self.dtype, self.is_cuda, self.device = dtype, True, "cuda:1"

    def get_device(self):
        return 1

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return A


@pytest.mark.parametrize("kv_dtype", ["fp8", "bf16", "fp4"])
@pytest.mark.parametrize("at", range(12))
def test_the_append_refuses_tensors_of_another_device(built_lib, monkeypatch, kv_dtype, at):
    import torch

    import glmkv
    from glmkv import ops

    monkeypatch.setattr(ops.torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops.torch, "Tensor", _OnDevice1)
    b, u, i = torch.bfloat16, torch.uint8, torch.int32
    names = [b, b, b, b, i, torch.int64, u, u, b, b, u, u]  # x, g_q, g_kv, rope, pos, slot, kv, idx, ik_w, ik_b, qq, qsf
    t = [A] * 12
    t[at] = _OnDevice1(names[at])
    with pytest.raises(ValueError, match="current device"):
        glmkv.mla_prep_full(t[0], 2752, *t[1:], 64, 64, kv_dtype=kv_dtype, stream=0)


def test_the_current_stream_without_torchs_private_name(monkeypatch):
    from types import SimpleNamespace

    from glmkv import ops

    monkeypatch.setattr(ops.torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(ops.torch.cuda, "current_stream", lambda: SimpleNamespace(cuda_stream=77))
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 100 + device)
    assert ops._stream(None) == 103
    monkeypatch.setattr(ops, "_raw_stream", None)
    monkeypatch.delattr(ops.torch._C, "_cuda_getCurrentRawStream", raising=False)
    assert ops._stream(None) == 77
    assert ops._stream(5) == 5 and ops._stream(SimpleNamespace(cuda_stream=6)) == 6


def test_plan_with_seen_checks_its_arguments(built_lib):
    import torch

    import glmkv
    from glmkv import _lib

    fn = glmkv.lib().glmkv_plan_seen
    good = [A, A, A, 2, A, A, A, A, A, A, 16, None]  # cu, seq_lens, seen, nseq, outputs, T, stream
    for i, v in [(3, 0), (10, -1)] + [(i, None) for i in (0, 1, 2, 4, 5, 6, 7, 8, 9)]:
        assert fn(*[v if j == i else a for j, a in enumerate(good)]) == _lib.ERR_ARG, (i, v)
    assert fn(*[0 if j == 10 else a for j, a in enumerate(good)]) == _lib.OK
    if not torch.cuda.is_available():
        with pytest.raises(glmkv.GlmKvError, match="glmkv_plan:"):
            glmkv.plan(A, A, 2, A, A, A, A, A, A, 16, stream=0)
        with pytest.raises(glmkv.GlmKvError, match="glmkv_plan_seen:"):
            glmkv.plan(A, A, 2, A, A, A, A, A, A, 16, stream=0, seen=A)


def test_launch_shapes_known_to_the_library(built_lib):
    """Every kernel that a cubin's user may launch has a shape (without a device: the query for it is reached); the
    eviction's, whose clusters follow from the call, are refused."""
    import torch

    import glmkv

    names = ["glm_mla_prep_fp4", "glm_kv4_dequant", "glm_kv4_attn", "glm_kv4_attn_picks", "glm_kv4_weights", "glm_kv4_join"]
    for name in names:
        if torch.cuda.is_available():
            assert min(glmkv.launch_shape(name, 8)[:2]) > 0
        else:
            with pytest.raises(glmkv.GlmKvError) as e:
                glmkv.launch_shape(name, 8)
            assert e.value.code == glmkv._lib.ERR_DEVICE, name
    assert glmkv.launch_shape("glm_plan_seen", 600) == glmkv.launch_shape("glm_plan", 600) == (3, 256, 0)
    for name in ("glm_evict_plan", "glm_evict_rows", "glm_evict_rows_fp4", "glm_evict_rows_fp8"):
        with pytest.raises(glmkv.GlmKvError, match="invalid argument"):
            glmkv.launch_shape(name, 8)
