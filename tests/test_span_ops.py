"""Step tables, windowed and shared-prefix attention: what the C ABI refuses before any launch, and the workspaces."""
import pytest
import torch

from ember_amd import _lib
from ember_amd import kernels as K


def _tables():
    a = _lib.StepTablesArgs()
    for f in ("cached_len", "new_len", "request_tables", "free_blocks", "query_start", "context_len", "positions", "token_seq",
              "slots", "block_tables", "totals"):
        setattr(a, f, 4096)  # never followed: every call here is refused
    a.S, a.R, a.max_blocks, a.n_free, a.max_tokens, a.pad_block = 2, 3, 4, 5, 6, 0
    return a


@pytest.mark.parametrize("field,value,text", [
    ("S", -1, "bad sizes"), ("S", _lib.STEP_MAX_SEQS + 1, "bad sizes"), ("R", -1, "bad sizes"), ("R", _lib.STEP_MAX_REQUESTS + 1, "bad sizes"),
    ("R", 1, "R must be at least S"), ("n_free", -1, "bad sizes"), ("max_tokens", -1, "bad sizes"), ("max_blocks", 0, "bad sizes"),
    ("max_blocks", 1 << 26, "31 bits"), ("pad_block", -2, "pad_block"), ("free_cursor", 4096 + 4, "free_cursor"),
    *((f, None, "null") for f in ("cached_len", "new_len", "request_tables", "free_blocks", "query_start", "context_len", "positions",
                                  "token_seq", "slots", "block_tables", "totals"))])
def test_step_tables_refusals(field, value, text):
    a = _tables()
    setattr(a, field, value)
    assert _lib.lib().ember_hip_step_tables(a, None) == _lib.ERR_INVALID
    assert text in _lib.last_error()


@pytest.mark.parametrize("field,at,other", [
    ("cached_len", 0x20000, "context_len"), ("request", 0x20000 + 4, "context_len"), ("new_len", 0x10000 + 8, "query_start"),
    ("request_tables", 0x60000 + 16, "block_tables"), ("free_blocks", 0x70000 - 4 * 4, "totals"), ("cached_len", 0x50000 + 44, "slots"),
    ("new_len", 0x30000 + 20, "positions"), ("request", 0x40000, "token_seq")])
def test_step_tables_refuse_to_work_in_place(field, at, other):
    """Inputs that overlap outputs, by one entry and more (S 2, R 3, 4 pages a row, 6 token rows); no pointer is followed."""
    a = _tables()
    for i, f in enumerate(("query_start", "context_len", "positions", "token_seq", "slots", "block_tables", "totals")):
        setattr(a, f, 0x10000 * (i + 1))
    for i, f in enumerate(("request", "cached_len", "new_len", "free_blocks", "request_tables")):
        setattr(a, f, 0x100000 + 0x10000 * i)
    setattr(a, field, at)
    assert _lib.lib().ember_hip_step_tables(a, None) == _lib.ERR_INVALID
    assert f"{field} overlaps {other}" in _lib.last_error()


def _batch(a):
    b = a  # the batch's fields come first
    for f in ("q", "k_cache", "v_cache", "out", "query_start", "positions", "block_tables"):
        setattr(b, f, 4096)
    b.T, b.S, b.max_blocks, b.n_heads, b.n_kv, b.head_dim, b.num_blocks = 4, 2, 8, 16, 8, 128, 32
    b.q_stride, b.scale, b.max_query, b.dtype = 2048, 0.1, 2, _lib.DTYPE_F16
    return a


def _window():
    a = _batch(_lib.WindowAttnArgs())
    a.window, a.sinks = 16, 4
    return a


def _prefix():
    a = _batch(_lib.PrefixAttnArgs())
    a.group_start, a.prefix_len, a.n_groups, a.max_group, a.max_prefix, a.max_own = 4096, 4096, 1, 4, 16, 16
    return a


BATCH = [("T", -1, "bad sizes"), ("S", -1, "bad sizes"), ("max_blocks", 0, "bad sizes"), ("max_blocks", 1 << 27, "bad sizes"),
         ("max_query", 0, "bad sizes"), ("n_heads", 15, "do not group"), ("n_kv", 0, "do not group"), ("head_dim", 64, "head_dim"),
         ("num_blocks", 0, "bad sizes"), ("dtype", 2, "dtype"), ("scale", 0.0, "scale"), ("scale", -1.0, "scale"),
         ("scale", float("nan"), "scale"), ("scale", float("inf"), "scale"), ("q_stride", 2040, "q_stride"), ("q_stride", 2052, "q_stride"),
         ("T", 1 << 28, "31 bits"), ("workspace", 8, "workspace"), ("workspace_bytes", -1, "workspace"), ("q", 4104, "aligned"),
         ("out", 4104, "aligned"), ("k_cache", 4104, "aligned"), ("v_cache", 4104, "aligned"),
         *((f, None, "null") for f in ("q", "k_cache", "v_cache", "out", "query_start", "positions", "block_tables"))]


@pytest.mark.parametrize("make,entry", [(_window, "ember_hip_window_attn"), (_prefix, "ember_hip_shared_prefix_attn")],
                         ids=["window", "prefix"])
@pytest.mark.parametrize("field,value,text", BATCH)
def test_batch_refusals(make, entry, field, value, text):
    a = make()
    setattr(a, field, value)
    assert getattr(_lib.lib(), entry)(a, None) == _lib.ERR_INVALID
    assert text in _lib.last_error()


@pytest.mark.parametrize("make,entry,field,value,text", [
    (_window, "ember_hip_window_attn", "window", 0, "window"), (_window, "ember_hip_window_attn", "sinks", -1, "sinks"),
    (_prefix, "ember_hip_shared_prefix_attn", "n_groups", -1, "bad sizes"), (_prefix, "ember_hip_shared_prefix_attn", "n_groups", 4097, "bad sizes"),
    (_prefix, "ember_hip_shared_prefix_attn", "max_group", 0, "bad sizes"), (_prefix, "ember_hip_shared_prefix_attn", "max_prefix", -1, "bad sizes"),
    (_prefix, "ember_hip_shared_prefix_attn", "max_own", 0, "bad sizes"), (_prefix, "ember_hip_shared_prefix_attn", "group_start", None, "null"),
    (_prefix, "ember_hip_shared_prefix_attn", "prefix_len", None, "null"), (_prefix, "ember_hip_shared_prefix_attn", "n_groups", 1, "bytes of workspace")])
def test_span_refusals(make, entry, field, value, text):
    a = make()
    setattr(a, field, value)
    assert getattr(_lib.lib(), entry)(a, None) == _lib.ERR_INVALID
    assert text in _lib.last_error()


def test_null_and_empty_calls():
    lib = _lib.lib()
    for entry in ("ember_hip_step_tables", "ember_hip_window_attn", "ember_hip_shared_prefix_attn"):
        assert getattr(lib, entry)(None, None) == _lib.ERR_INVALID
    for entry in ("ember_hip_window_workspace_bytes", "ember_hip_shared_prefix_workspace_bytes"):
        assert getattr(lib, entry)(None) == 0
    for make, entry in ((_window, "ember_hip_window_attn"), (_prefix, "ember_hip_shared_prefix_attn")):
        for field in ("T", "S"):
            a = make()
            setattr(a, field, 0)
            assert getattr(lib, entry)(a, None) == _lib.OK  # nothing to do, nothing launched


def test_workspace_covers_smaller_tables():
    """A workspace sized without a table width holds the partials of any table width."""
    size = _lib.lib().ember_hip_window_workspace_bytes
    for S in (1, 3, 40):
        for window in (20, 500, 5000):
            for q in (1, 9, 200):
                a = _window()
                a.window, a.S, a.T, a.max_query, a.max_blocks = window, S, S * q, q, 1 << 26
                most = size(a)
                for blocks in (1, 7, 33, 64, 130, 400, 1000):
                    a.max_blocks = blocks
                    assert size(a) <= most
    assert K.window_workspace(4, 4, n_heads=16, n_kv=8, window=100000, max_query=1, device="cpu") is not None
    assert K.window_workspace(1, 1, n_heads=16, n_kv=8, window=10, max_query=1, device="cpu") is None


def test_a_window_workspace_covers_smaller_batches():
    """Fewer sequences split more: what one of them needs alone, a larger batch's workspace holds."""
    size = _lib.lib().ember_hip_window_workspace_bytes

    def bytes_for(S, q, **kw):
        a = _window()
        a.window, a.S, a.T, a.max_query, a.max_blocks = 4096, S, S * q, q, 1 << 26
        for k, v in kw.items():
            setattr(a, k, v)
        return size(a)
    for kw in (dict(), dict(dtype=_lib.DTYPE_F32), dict(n_heads=8, n_kv=1, q_stride=1024)):
        for q in (1, 4, 300):
            sizes = [bytes_for(S, q, **kw) for S in (1, 2, 5, 16, 33, 100, 400)]
            assert sizes == sorted(sizes) and sizes[0] > 0
            assert bytes_for(7, 1, **kw) <= bytes_for(7, q, **kw)


@pytest.mark.parametrize("make,entry", [(_window, "ember_hip_window_attn"), (_prefix, "ember_hip_shared_prefix_attn")],
                         ids=["window", "prefix"])
def test_more_sequences_than_one_launch_holds_are_refused(make, entry):
    """2^24 work-groups of 256 threads are 2^32 threads; no pointer is followed."""
    a = make()
    a.S, a.max_query, a.workspace, a.workspace_bytes = 1 << 21, 1, 4096, 1 << 40
    assert getattr(_lib.lib(), entry)(a, None) == _lib.ERR_INVALID
    assert "too many work-groups" in _lib.last_error()


def test_a_window_workspace_covers_padded_batches():
    """The same with rows of padding: T stays, or shrinks less than the sequences and their tokens do."""
    size = _lib.lib().ember_hip_window_workspace_bytes
    for kw in (dict(), dict(dtype=_lib.DTYPE_F32), dict(n_heads=8, n_kv=1, q_stride=1024)):
        for T, S, q in ((512, 512, 1), (512, 64, 8), (64, 64, 1), (2048, 4, 512), (300, 1, 300)):
            def bytes_for(t, s, m, blocks=1 << 26):
                a = _window()
                a.window, a.T, a.S, a.max_query, a.max_blocks = 4096, t, s, m, blocks
                for k, v in kw.items():
                    setattr(a, k, v)
                return size(a)
            most = bytes_for(T, S, q)
            for t in (T, T // 2 + 1, 1):
                for s in {S, S // 2 + 1, 4, 1}:
                    for m in {q, q // 3 + 1, 2, 1}:
                        for blocks in (1 << 26, 100, 3):
                            if s <= S and m <= q:
                                assert bytes_for(t, s, m, blocks) <= most, (kw, T, S, q, t, s, m, blocks)


APART = {f: 0x10000 * (i + 1) for i, f in enumerate(
    ("query_start", "context_len", "positions", "token_seq", "slots", "block_tables", "totals", "request", "cached_len", "new_len",
     "free_blocks", "free_cursor", "request_tables"))}


@pytest.mark.parametrize("field,at,text", [
    # the request tables are written, beside every other input (3 rows of 4 pages)
    ("request", APART["request_tables"] + 44, "request overlaps request_tables"), ("cached_len", APART["request_tables"] - 8, "cached_len overlaps request_tables"),
    ("new_len", APART["request_tables"] + 16, "new_len overlaps request_tables"), ("free_blocks", APART["request_tables"] + 20, "free_blocks overlaps request_tables"),
    ("free_cursor", APART["request_tables"] + 40, "free_cursor overlaps request_tables"),
    # the cursor in any output
    ("free_cursor", APART["query_start"] + 8, "free_cursor overlaps query_start"), ("free_cursor", APART["context_len"], "free_cursor overlaps context_len"),
    ("free_cursor", APART["positions"] + 20, "free_cursor overlaps positions"), ("free_cursor", APART["slots"] + 44, "free_cursor overlaps slots"),
    ("free_cursor", APART["block_tables"], "free_cursor overlaps block_tables"), ("free_cursor", APART["totals"] + 4, "free_cursor"),
    # two outputs
    ("positions", APART["token_seq"] + 20, "positions overlaps token_seq"), ("context_len", APART["query_start"] + 8, "query_start overlaps context_len"),
    ("request_tables", APART["slots"] + 40, "request_tables overlaps slots"), ("totals", APART["block_tables"] + 44, "block_tables overlaps totals")])
def test_step_tables_refuse_what_another_work_group_would_write(field, at, text):
    a = _tables()
    for f, x in APART.items():
        setattr(a, f, x)
    setattr(a, field, at)
    assert _lib.lib().ember_hip_step_tables(a, None) == _lib.ERR_INVALID
    assert text in _lib.last_error()


@pytest.mark.parametrize("make,entry", [(_window, "ember_hip_window_attn"), (_prefix, "ember_hip_shared_prefix_attn")],
                         ids=["window", "prefix"])
def test_scales_that_are_infinite_in_base_2_are_refused(make, entry):
    a = make()
    a.scale = 3e38
    assert getattr(_lib.lib(), entry)(a, None) == _lib.ERR_INVALID
    assert "scale" in _lib.last_error()


@pytest.mark.parametrize("bad", [dict(n_heads=15), dict(n_kv=0), dict(T=-1), dict(S=-2), dict(max_query=0), dict(max_blocks=0),
                                 dict(dtype=torch.bfloat16), dict(dtype=torch.int32)])
@pytest.mark.parametrize("make", [K.window_workspace, K.shared_prefix_workspace], ids=["window", "prefix"])
def test_workspaces_of_sizes_that_no_call_takes_are_refused(make, bad):
    kw = dict(T=64, S=8, n_heads=16, n_kv=8, max_query=8, device="cpu")
    kw.update(dict(window=4096) if make is K.window_workspace else dict(n_groups=2))
    assert make(**kw) is not None
    with pytest.raises(K.EmberError):
        make(**{**kw, **bad})
    assert make(**{**kw, "T": 0}) is None
