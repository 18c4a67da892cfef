"""A cache and weights in 4 bits: the format's reference, and what the C ABI refuses before any launch."""
import numpy as np
import pytest
import torch

import four_bit_reference as ref
from ember_amd import _lib
from ember_amd import kernels as K


def test_reference_codes_are_nearest_and_scales_lowest(rng):
    x = rng.standard_normal((50, 64)) * 2.0 ** rng.integers(-20, 12, (50, 1))
    x[0], x[1, :32], x[2, :32] = 0, 7.0, np.nextafter(7.0, 8)
    code, scale = ref.encode(x)
    back = ref.decode(code, scale)
    unit = np.repeat(2.0 ** (scale.astype(float) - 127), 32, -1)
    assert (np.abs(back - x) <= unit * np.where(np.abs(x) > 4 * unit, 1, np.where(np.abs(x) > 2 * unit, 0.5, 0.25))).all()
    assert (np.abs(x).reshape(50, 2, 32).max(-1) > 3.5 * 2.0 ** (scale.astype(float) - 127))[1:].all()
    assert scale[1, 0] == 127 and scale[2, 0] == 128 and (scale[0] == 104).all()
    assert (back[1, :32] == 6).all()
    # ties go to the even code
    t = np.zeros((1, 32))
    t[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5]
    t[0, 31] = 6
    assert ref.encode(t)[0][0, :8].tolist() == [0, 2, 2, 4, 4, 6, 6, 14]


def test_reference_pages_go_both_ways(rng):
    k, v = rng.standard_normal((2, 3, 2, 16, 128))
    pages = ref.to_pages(k, v)
    assert pages.shape == (3, 2, K.KV4_PAGE_BYTES) == (3, 2, ref.PAGE_BYTES)
    one = np.zeros_like(pages)
    for n in range(3):
        for h in range(2):
            for s in range(16):
                ref.write_slot(one[n, h], s, k[n, h, s], v[n, h, s])
    assert np.array_equal(one, pages)
    kk, vv = ref.read_pages(pages)
    assert np.array_equal(kk, ref.decode(*ref.encode(k))) and np.array_equal(vv, ref.decode(*ref.encode(v)))


def _append():
    a = _lib.Kv4AppendArgs()
    for f in ("qkv", "q_out", "pool", "inv_freq", "positions", "token_seq", "block_tables"):
        setattr(a, f, 4096)  # never followed: every call here is refused
    a.rows, a.max_blocks, a.T, a.n_heads, a.n_kv, a.head_dim, a.num_blocks, a.eps = 3, 4, 5, 16, 8, 128, 6, 1e-6
    return a


@pytest.mark.parametrize("field,value,text", [
    ("head_dim", 64, "head_dim"), ("n_heads", 15, "do not group"), ("n_heads", 128, "at most 64"), ("n_kv", 0, "do not group"),
    ("T", -1, "bad sizes"), ("T", 1 << 24, "bad sizes"), ("rows", 0, "bad sizes"), ("max_blocks", 0, "bad sizes"), ("num_blocks", 0, "bad sizes"),
    ("q_norm", 4096, "go together"), ("k_norm", 4096, "go together"), ("k_out", 4096, "go together"), ("v_out", 4096, "go together"),
    ("qkv", 4104, "aligned"), ("q_out", 4104, "aligned"), ("pool", 4104, "aligned"),
    *((f, None, "null") for f in ("qkv", "q_out", "pool", "inv_freq", "positions", "token_seq", "block_tables"))])
def test_append_refusals(field, value, text):
    a = _append()
    setattr(a, field, value)
    assert _lib.lib().ember_hip_kv4_append(a, None) == _lib.ERR_INVALID
    assert text in _lib.last_error()


def test_calls_without_tokens_do_nothing():
    a = _append()
    a.T = 0
    assert _lib.lib().ember_hip_kv4_append(a, None) == _lib.OK
    for f in ("T", "S"):
        b = _attn()
        setattr(b, f, 0)
        assert _lib.lib().ember_hip_kv4_attn(b, None) == _lib.OK
        assert _lib.lib().ember_hip_kv4_workspace_bytes(b) == 0 and _lib.last_error() == ""
    g = _gemv()
    g.M = 0
    assert _lib.lib().ember_hip_gemv4(g, None) == _lib.OK
    q = _quantize()
    q.rows = 0
    assert _lib.lib().ember_hip_mx_quantize(q, None) == _lib.OK


def _attn():
    a = _lib.Kv4AttnArgs()
    for f in ("q", "k_cache", "out", "query_start", "positions", "block_tables"):
        setattr(a, f, 4096)
    a.T, a.S, a.max_blocks, a.n_heads, a.n_kv, a.head_dim, a.num_blocks = 4, 2, 8, 16, 8, 128, 32
    a.q_stride, a.scale, a.max_query, a.dtype, a.max_context = 2048, 0.1, 2, _lib.DTYPE_F16, 100
    return a


SIZES = [("T", -1, "bad sizes"), ("S", -1, "bad sizes"), ("max_blocks", 0, "bad sizes"), ("max_blocks", 1 << 27, "bad sizes"),
         ("max_query", 0, "bad sizes"), ("n_heads", 15, "do not group"), ("n_kv", 0, "do not group"), ("head_dim", 64, "head_dim"),
         ("dtype", 2, "dtype"), ("dtype", _lib.DTYPE_F32, "f16"), ("T", 1 << 28, "31 bits"), ("max_context", 0, "max_context"),
         ("max_context", -1, "max_context"), ("v_cache", 4096, "v_cache")]


@pytest.mark.parametrize("field,value,text", SIZES + [
    ("num_blocks", 0, "bad sizes"), ("scale", 0.0, "scale"), ("scale", -1.0, "scale"), ("scale", float("nan"), "scale"),
    ("scale", float("inf"), "scale"), ("scale", 3e38, "scale"), ("q_stride", 2040, "q_stride"), ("q_stride", 2052, "q_stride"),
    ("workspace", 8, "workspace"), ("workspace_bytes", -1, "workspace"), ("q", 4104, "aligned"), ("out", 4104, "aligned"),
    ("k_cache", 4104, "aligned"), *((f, None, "null") for f in ("q", "k_cache", "out", "query_start", "positions", "block_tables"))])
def test_attention_refusals(field, value, text):
    a = _attn()
    setattr(a, field, value)
    assert _lib.lib().ember_hip_kv4_attn(a, None) == _lib.ERR_INVALID
    assert text in _lib.last_error()


@pytest.mark.parametrize("field,value,text", SIZES)
def test_workspaces_refuse_sizes_that_no_call_takes(field, value, text):
    a = _attn()
    setattr(a, field, value)
    assert _lib.lib().ember_hip_kv4_workspace_bytes(a) == 0
    assert text in _lib.last_error()


def test_attention_refuses_launches_that_are_too_large():
    a = _attn()
    a.T, a.S, a.n_kv, a.n_heads, a.max_query = 1 << 12, 4096, 1 << 15, 1 << 15, 512
    a.q_stride = 128 << 15
    assert _lib.lib().ember_hip_kv4_attn(a, None) == _lib.ERR_INVALID
    assert "work-groups" in _lib.last_error()


def _quantize():
    a = _lib.MxQuantizeArgs()
    a.x, a.codes, a.scales, a.ld, a.rows, a.cols, a.dtype = 4096, 4096, 4096, 64, 2, 64, _lib.DTYPE_F16
    return a


@pytest.mark.parametrize("field,value,text", [
    ("rows", -1, "multiple of 32"), ("cols", -32, "multiple of 32"), ("cols", 48, "multiple of 32"), ("ld", 63, "ld at least"),
    ("dtype", 2, "dtype"), ("x", None, "null"), ("codes", None, "null"), ("scales", None, "null"), ("x", 4097, "aligned"),
    ("codes", 4098, "aligned")])
def test_quantize_refusals(field, value, text):
    a = _quantize()
    setattr(a, field, value)
    assert _lib.lib().ember_hip_mx_quantize(a, None) == _lib.ERR_INVALID
    assert text in _lib.last_error()


@pytest.mark.parametrize("N,k", [(0, 64), (-1, 64), (16, 0), (16, 48), (16, -32), ((1 << 24) + 1, 32), (16, (1 << 24) + 32)])
def test_weight_sizes_refused(N, k):
    lib = _lib.lib()
    assert lib.ember_hip_gemv4_packed_bytes(N, k) == 0 and "multiple of 32" in _lib.last_error()
    assert lib.ember_hip_gemv4_pack(4096, 4096, N, k, 4096, None) == _lib.ERR_INVALID
    g = _gemv()
    g.N, g.K = N, k
    assert lib.ember_hip_gemv4(g, None) == _lib.ERR_INVALID and "multiple of 32" in _lib.last_error()


@pytest.mark.parametrize("args,text", [((None, 4096, 4096), "null"), ((4096, None, 4096), "null"), ((4096, 4096, None), "null"),
                                       ((4098, 4096, 4096), "aligned"), ((4096, 4096, 4104), "aligned")])
def test_pack_refusals(args, text):
    assert _lib.lib().ember_hip_gemv4_pack(args[0], args[1], 16, 32, args[2], None) == _lib.ERR_INVALID
    assert text in _lib.last_error()


def test_packed_sizes():
    f = _lib.lib().ember_hip_gemv4_packed_bytes
    assert f(16, 128) == f(1, 32) == 1088 and f(17, 129 * 32) == 2 * 33 * 1088


def _gemv():
    g = _lib.Gemv4Args()
    g.A, g.W, g.C, g.lda, g.ldc, g.M, g.N, g.K, g.epilogue = 4096, 4096, 4096, 64, 32, 2, 32, 64, 0
    return g


@pytest.mark.parametrize("field,value,text", [
    ("M", -1, "M must be"), ("M", (1 << 21) + 1, "M must be"), ("epilogue", 4, "epilogue"), ("epilogue", -1, "epilogue"), ("lda", 56, "lda"),
    ("lda", 68, "lda"), ("ldc", 31, "ldc"), ("A", None, "null"), ("W", None, "null"), ("C", None, "null"), ("A", 4104, "aligned"),
    ("W", 4104, "aligned"), ("C", 4097, "aligned")])
def test_gemv_refusals(field, value, text):
    g = _gemv()
    setattr(g, field, value)
    assert _lib.lib().ember_hip_gemv4(g, None) == _lib.ERR_INVALID
    assert text in _lib.last_error()


def test_gemv_refuses_half_pairs_and_misaligned_floats():
    g = _gemv()
    g.N, g.epilogue = 31, _lib.EPILOGUE_SILU_MUL
    assert _lib.lib().ember_hip_gemv4(g, None) == _lib.ERR_INVALID and "even N" in _lib.last_error()
    g.N, g.epilogue, g.C = 32, _lib.EPILOGUE_ADD_F32, 4098
    assert _lib.lib().ember_hip_gemv4(g, None) == _lib.ERR_INVALID and "aligned" in _lib.last_error()


@pytest.mark.parametrize("call", [
    lambda h: K.kv4_append(h, h, h, h, h, h, n_heads=1, n_kv=1, inv_freq_dev=h),
    lambda h: K.kv4_attention(h.view(1, 1, 128), h, h, h, h, h),
    lambda h: K.mx_quantize(h.view(1, 128)),
    lambda h: K.gemv4_pack(h.view(torch.uint8).view(2, 128), h.view(torch.uint8).view(2, 128)),
    lambda h: K.gemv4(h.view(1, 128), h, h, 0, N=16)])
def test_python_refuses_host_tensors(call):
    with pytest.raises(_lib.EmberError):
        call(torch.zeros(128, dtype=torch.float16))


def test_python_refuses_contexts_and_workspace_sizes():
    with pytest.raises(_lib.EmberError, match="max_context"):
        K.kv4_workspace(4, 2, n_heads=16, n_kv=8, max_context=0, device="cpu")
    with pytest.raises(_lib.EmberError, match="do not group"):
        K.kv4_workspace(4, 2, n_heads=15, n_kv=8, max_context=10, device="cpu")
    assert K.kv4_workspace(4, 2, n_heads=16, n_kv=8, max_context=16, device="cpu") is None


def test_workspaces_are_enough_for_smaller_batches(rng):
    size = _lib.lib().ember_hip_kv4_workspace_bytes
    for _ in range(300):
        n_kv, G = int(rng.choice([1, 2, 8])), int(rng.choice([1, 2, 3, 4, 8]))
        S, mq, ctx = (int(2 ** rng.uniform(0, x)) for x in (9, 11, 17))
        T = min(S * mq, 1 << 14)

        def need(T, S, mq, ctx):
            a = _lib.Kv4AttnArgs()
            a.T, a.S, a.max_blocks, a.n_heads, a.n_kv, a.head_dim, a.dtype = T, S, 1 << 14, n_kv * G, n_kv, 128, _lib.DTYPE_F16
            a.max_query, a.max_context = mq, ctx
            return size(a)
        most = need(T, S, mq, ctx)
        for _ in range(8):
            less = [max(1, int(x * rng.uniform(0, 1))) for x in (T, S, mq, ctx)]
            assert need(*less) <= most, (T, S, mq, ctx, less)


def _plan(T, S, n_heads, n_kv, max_query, max_context, max_blocks=1 << 14, workspace_bytes=1 << 40):
    """The launches of a call of these sizes, as a list."""
    a = _attn()
    a.T, a.S, a.n_heads, a.n_kv, a.max_query, a.max_context, a.max_blocks = T, S, n_heads, n_kv, max_query, max_context, max_blocks
    a.workspace, a.workspace_bytes = (4096, workspace_bytes) if workspace_bytes else (None, 0)  # not followed
    out = (_lib.Kv4Launch * 2)()
    n = _lib.lib().ember_hip_kv4_attn_plan(a, out)
    assert n >= 0, _lib.last_error()
    return list(out[:n])


@pytest.mark.parametrize("field,value,text", SIZES)
def test_plans_refuse_sizes_that_no_call_takes(field, value, text):
    a = _attn()
    setattr(a, field, value)
    assert _lib.lib().ember_hip_kv4_attn_plan(a, (_lib.Kv4Launch * 2)()) == _lib.ERR_INVALID
    assert text in _lib.last_error()


def test_plans_of_nothing():
    lib, out = _lib.lib(), (_lib.Kv4Launch * 2)()
    assert lib.ember_hip_kv4_attn_plan(None, out) == _lib.ERR_INVALID and "null" in _lib.last_error()
    assert lib.ember_hip_kv4_attn_plan(_attn(), None) == _lib.ERR_INVALID and "null" in _lib.last_error()
    assert _plan(0, 2, 16, 8, 1, 100) == _plan(4, 0, 16, 8, 1, 100) == []


def test_plans_of_the_forms():
    """One sequence's decode, runs of up to 32 rows, prompts, many decodes, a step of decodes and a few chunks."""
    one = _plan(1, 1, 16, 8, 1, 640)
    assert [(x.rows, x.sharers, x.dealt) for x in one] == [(16, 0, 0)]
    assert [(x.rows, x.sharers > 0) for x in _plan(1, 1, 16, 8, 1, 131072)] == [(16, True)]
    assert [x.rows for x in _plan(20, 5, 32, 8, 8, 640)] == [32] and [x.rows for x in _plan(20, 5, 32, 8, 9, 640)] == [128]
    assert [(x.rows, x.sharers, x.dealt) for x in _plan(64, 64, 16, 8, 1, 4096)] == [(16, 0, 1)]
    mixed = _plan(960 + 40 * 512, 1000, 16, 8, 512, 1512)
    assert [(x.rows, x.least, x.most) for x in mixed] == [(16, 1, 16), (128, 17, 2 ** 31 - 1)]
    # without a workspace nothing is shared, with too small a one neither
    for size in (0, mixed[1].workspace - 1):
        assert all(x.sharers == 0 for x in _plan(960 + 40 * 512, 1000, 16, 8, 512, 1512, workspace_bytes=size))


def test_workspaces_are_enough_for_what_their_calls_launch(rng):
    """The reported size, whose launches' rows are not known yet, against what every launch of a call asks for."""
    seen = set()
    for _ in range(3000):
        n_kv, G = int(rng.choice([1, 2, 8])), int(rng.choice([1, 2, 3, 4, 8, 16, 20, 32, 40]))
        S, mq, ctx, W = (int(2 ** rng.uniform(0, x)) for x in (11, 11, 17, 13))
        T = min(int(S * mq * rng.uniform(0, 1)) + 1, 1 << 16)
        a = _attn()
        a.T, a.S, a.max_blocks, a.n_heads, a.n_kv, a.max_query, a.max_context = T, S, W, n_kv * G, n_kv, mq, ctx
        size = _lib.lib().ember_hip_kv4_workspace_bytes(a)
        less = [max(1, int(x * rng.uniform(0, 1))) for x in (T, S, mq, ctx)]
        for t, s, q, c in ((T, S, mq, ctx), less):
            plan = _plan(t, s, n_kv * G, n_kv, q, c, W)
            assert all(x.workspace <= size for x in plan), (T, S, mq, ctx, W, n_kv, G, t, s, q, c)
            seen |= {(len(plan), x.rows, x.sharers > 0, x.dealt) for x in plan}
    # of every kind: in one launch and in two, each form, shared and not, dealt
    assert {(1, r, cut, 0) for r in (16, 32, 128) for cut in (False, True)} <= seen
    assert {(2, 16, True, 0), (2, 128, True, 0), (1, 16, False, 1), (1, 32, False, 1)} <= seen


@pytest.mark.parametrize("G,few", [(1, 16), (16, 16), (17, 32), (20, 32), (32, 32), (33, 0), (40, 0)])
def test_no_launch_of_a_mixed_step_is_for_rows_that_no_sequence_has(G, few):
    """A sequence has the rows of one token at least: short ones are walked, up to 32 rows where a token has more than 16."""
    got = [(x.rows, x.least, x.most) for x in _plan(70 + 200, 72, 2 * G, 2, 130, 30_000)]
    tiles = (128, few + 1, 2 ** 31 - 1)
    assert got == ([(few, 1, few), tiles] if few else [tiles])
