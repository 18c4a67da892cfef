"""Step tables, windowed attention and shared-prefix attention on the GPU, against plain Python / float64 references.

Slots that no token may see hold NaN (values and keys), pages that are not needed are -1 in the tables or hold NaN,
and rows that belong to no sequence must keep what they held. Bounds are derived in span_reference.
"""
import ctypes

import numpy as np
import pytest
import torch

from ember_amd import _lib
from ember_amd import kernels as K
from ember_amd._lib import EmberError
from span_reference import D, PAGE, attention_reference, step_tables_reference

pytestmark = pytest.mark.gpu


def dint(a, device):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)


# ---- step tables ----

FIELDS = ("query_start", "context_len", "positions", "token_seq", "slots", "block_tables", "totals")


def run_tables(device, request, cached, new, tables, free, cursor, max_tokens, pad):
    out = K.StepTables(len(new), max_tokens, tables.shape[1], device)
    for f in FIELDS:
        getattr(out, f).fill_(-77)
    rt = dint(tables, device)
    args = (out, rt, dint(cached, device), dint(new, device), dint(free, device))
    kw = dict(request=None if request is None else dint(request, device),
              free_cursor=None if cursor is None else dint([cursor], device), pad_block=pad)
    for _ in range(2):  # a repeated call gives the same
        K.step_tables(*args, **kw)
    torch.cuda.synchronize()
    got = {f: getattr(out, f).cpu().numpy() for f in FIELDS}
    got["request_tables"] = rt.cpu().numpy()
    return got


def check_tables(device, request, cached, new, tables, free, cursor, max_tokens, pad):
    want = step_tables_reference(request, cached, new, tables, free, cursor or 0, max_tokens, pad)
    got = run_tables(device, request, cached, new, tables, free, cursor, max_tokens, pad)
    for f in want:
        assert np.array_equal(got[f], want[f]), f
    return want["totals"]


def random_tables(rng, S, R, W, top_cached, top_new, short=0):
    request = rng.permutation(R)[:S]
    cached = rng.integers(0, top_cached + 1, R)
    new = rng.integers(0, top_new + 1, S)
    place = rng.permutation(R * W + 64)
    tables = np.full((R, W), -1)
    for r in range(R):
        n = min(W, -(-int(cached[r]) // PAGE))
        tables[r, :n] = place[r * W:r * W + n]
    need = sum(-(-int(c + n) // PAGE) - -(-int(c) // PAGE) for c, n in zip(cached[request], new))
    free = rng.permutation(10 * R * W + 100)[:max(0, need - short)]
    return request, cached, new, tables, free


@pytest.mark.parametrize("S,R,W,top_cached,top_new", [
    (1, 1, 1, 0, 1), (1, 3, 4, 30, 20), (7, 9, 13, 150, 40), (64, 64, 16, 200, 3), (33, 100, 1030, 16000, 300),
    (300, 300, 8, 100, 1), (257, 1000, 64, 900, 100)])
def test_step_tables_match_the_reference(rng, device, S, R, W, top_cached, top_new):
    request, cached, new, tables, free = random_tables(rng, S, R, W, top_cached, top_new)
    T = int(new.sum())
    assert check_tables(device, request, cached, new, tables, free, 0, T + 5, 3)[2] == 0
    front = np.concatenate([np.full(3, 9999), free])  # three entries taken by earlier steps
    check_tables(device, request, cached, new, tables, front, 3, T, -1)


def test_step_tables_without_request_list(rng, device):
    _, cached, new, tables, free = random_tables(rng, 6, 6, 12, 120, 30)
    check_tables(device, None, cached, new[:6], tables, np.arange(1000, 1100), None, 400, 7)


def test_step_tables_refuse_what_cannot_be_placed(rng, device):
    """Each refusal sets its bit and leaves the others' tokens where they belong."""
    request, cached, new, tables, free = random_tables(rng, 40, 50, 20, 250, 40)
    T = int(new.sum())
    assert check_tables(device, request, cached, new, tables, free, 0, T // 2, 0)[2] & _lib.STEP_LATE
    assert check_tables(device, request, cached, new, tables, free[: len(free) // 2], 0, T, 0)[2] & _lib.STEP_SHORT
    assert check_tables(device, request, cached, new, tables, free[:0], 0, T, 0)[2] & _lib.STEP_SHORT
    assert check_tables(device, request, cached, new, tables, free[: len(free) // 2], 2, T // 2, 0)[2]
    assert check_tables(device, request, cached, new, tables, free, len(free) + 9, T, 0)[2] & _lib.STEP_SHORT
    check_tables(device, request, cached, new, tables, free, -5, T, 0)
    wide = new.copy()
    wide[3], wide[17] = 20 * PAGE + 1, 2 ** 31 - 1
    assert check_tables(device, request, cached, wide, tables, free, 0, T, 0)[2] & _lib.STEP_WIDE
    twice = request.copy()
    twice[5] = twice[30] = twice[31]
    twice[8], twice[9] = -1, 50
    bad = new.copy()
    bad[11] = -3
    long = cached.copy()
    long[request[12]], long[request[13]] = 20 * PAGE + 1, -1
    assert check_tables(device, twice, long, bad, tables, free, 0, T, 0)[2] & _lib.STEP_INVALID


def test_step_tables_exact_fits_and_no_sequences(rng, device):
    # contexts that end on a page, and tables filled to the last entry
    tables = np.arange(24).reshape(3, 8)
    cached, new = np.array([16, 112, 0]), np.array([16, 16, 128])
    tables[0, 1:] = tables[1, 7:] = tables[2, :] = -1
    assert check_tables(device, None, cached, new, tables, np.arange(100, 110), 0, 160, 5)[2] == 0
    check_tables(device, None, np.zeros(0, int), np.zeros(0, int), np.zeros((0, 4), int), np.arange(3), 1, 70, 5)
    check_tables(device, None, np.array([5]), np.array([0]), np.array([[2, -1]]), np.zeros(0, int), None, 0, -1)


def test_step_tables_largest_batch(rng, device):
    request, cached, new, tables, free = random_tables(rng, 4096, 65536, 4, 60, 3)
    ok = cached[request] + new <= 64
    new = np.where(ok, new, 0)
    assert check_tables(device, request, cached, new, tables, free, 0, int(new.sum()) + 100, 1)[2] == 0


def test_step_tables_python_refusals(device):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)  # noqa: E731
    out = K.StepTables(2, 8, 4, device)
    good = (i(3, 4), i(3), i(2), i(5))
    for at, bad in ((0, i(3, 5)), (0, i(3, 8)[:, ::2]), (0, i(3, 4).long()), (1, i(2)), (2, i(3)), (3, i(5, 1)),
                    (1, torch.zeros(3, dtype=torch.int32)), (3, i(10)[::2])):
        args = list(good)
        args[at] = bad
        with pytest.raises(EmberError):
            K.step_tables(out, *args)
    with pytest.raises(EmberError):
        K.step_tables(out, *good, request=i(3))
    with pytest.raises(EmberError):
        K.step_tables(out, *good, free_cursor=out.totals[1:2])
    with pytest.raises(EmberError, match="cached_len overlaps context_len"):
        K.step_tables(out, i(2, 4), out.context_len, i(2), i(5))
    with pytest.raises(EmberError, match="request_tables overlaps block_tables"):
        K.step_tables(out, out.block_tables, i(3), i(2), i(5))
    with pytest.raises(EmberError):
        K.step_tables(out, *good, pad_block=-2)
    with pytest.raises(EmberError):
        K.step_tables(out, i(1, 4), i(1), i(2), i(5))  # two sequences, one request row, no list
    with pytest.raises(EmberError):
        K.StepTables(2, 8, 4, "cpu")


# ---- the two attentions ----

class Batch:
    """A ragged batch over scattered pages. need(s, j): whether some token of sequence s sees key j; every slot that
    is not needed holds NaN, and a page without a needed slot is -1 in the table (or, `stale`, a page of NaN)."""

    def __init__(self, rng, device, cached, new, heads, kv, f16, need, *, shared=None, stale=False, pad_rows=3, spread=1.5):
        self.cached, self.new = np.asarray(cached), np.asarray(new)
        S = self.cached.size
        ctx = self.cached + self.new
        self.start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int64)
        T = int(self.start[-1])
        self.pos = np.concatenate([np.arange(c, c + n) for c, n in zip(self.cached, self.new)] + [np.zeros(0, int)])
        W = max(1, int(-(-ctx.max() // PAGE)) + 2)
        blocks = int((-(-ctx // PAGE)).sum()) + 9
        place = rng.permutation(blocks)
        nan_page, place = place[0], place[1:]
        self.tables = np.full((S, W), -1)
        dt = np.float16 if f16 else np.float32
        k = np.full((blocks, kv, PAGE, D), np.nan, dt)
        v = k.copy()
        at = 0
        for s in range(S):
            first, upto = (0, 0) if shared is None else shared(s)  # whole pages of sequence `first` up to key `upto`
            for pg in range(-(-int(ctx[s]) // PAGE)):
                j = np.arange(pg * PAGE, min((pg + 1) * PAGE, ctx[s]))
                if first != s and (pg + 1) * PAGE <= upto:
                    self.tables[s, pg] = self.tables[first, pg]
                    continue
                live = j[need(s, j)]
                if not live.size:
                    self.tables[s, pg] = nan_page if stale else -1
                    continue
                b = place[at]
                at += 1
                self.tables[s, pg] = b
                k[b, :, live % PAGE] = rng.standard_normal((live.size, kv, D)).astype(dt)
                v[b, :, live % PAGE] = rng.standard_normal((live.size, kv, D)).astype(dt)
                if first != s and pg * PAGE < upto:  # the shared part of a partly shared page is a copy
                    n = upto - pg * PAGE
                    src = self.tables[first, pg]
                    k[b, :, :n], v[b, :, :n] = k[src, :, :n], v[src, :, :n]
        self.k, self.v = k, v
        self.q = (spread * rng.standard_normal((T + pad_rows, heads, D))).astype(dt)
        self.T, self.f16 = T, f16
        self.dev = dict(q=torch.from_numpy(self.q).to(device), k=torch.from_numpy(k).to(device),
                        v=torch.from_numpy(v).to(device), start=dint(self.start, device),
                        pos=dint(np.concatenate([self.pos, np.full(pad_rows, 7)]), device), table=dint(self.tables, device))
        self.out = torch.full((T + pad_rows, heads, D), 123.0, dtype=torch.float16 if f16 else torch.float32, device=device)

    def args(self):
        d = self.dev
        return d["q"], d["k"], d["v"], self.out, d["start"], d["pos"], d["table"]

    def check(self, sees):
        torch.cuda.synchronize()
        got = self.out.double().cpu().numpy()
        assert (got[self.T:] == 123.0).all(), "rows of no sequence were written"
        want, bound = attention_reference(self.q[:self.T], self.k, self.v, self.tables, self.start, self.pos, sees, self.f16)
        off = np.abs(got[:self.T] - want)
        assert np.isfinite(got).all()
        worst = (off - bound).max() if off.size else 0
        assert worst <= 0, f"off by {off.max():.3e}, beyond its bound by {worst:.3e}"
        return got[:self.T]


def window_batch(rng, device, cached, new, heads, kv, f16, window, sinks, **kw):
    sees = lambda s, p, j: (j <= p) & ((p - j < window) | (j < sinks))  # noqa: E731
    lo = lambda s: int(cached[s]) - window + 1  # noqa: E731
    b = Batch(rng, device, cached, new, heads, kv, f16, lambda s, j: (j >= lo(s)) | (j < sinks), **kw)
    return b, sees


def window_ws(b, heads, kv, window, sinks, device, max_query=None):
    return K.window_workspace(b.q.shape[0], b.cached.size, n_heads=heads, n_kv=kv, window=window, sinks=sinks,
                              max_query=max_query, dtype=torch.float16 if b.f16 else torch.float32, device=device)


CONTEXTS = [0, 1, 15, 16, 17, 40, 130, 300, 700]


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("heads,kv", [(2, 2), (16, 8), (6, 2), (8, 1), (20, 2)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 0), (100, 33), (1000, 5)])
def test_window_decode(rng, device, f16, heads, kv, window, sinks):
    new = np.ones(len(CONTEXTS), int)
    b, sees = window_batch(rng, device, CONTEXTS, new, heads, kv, f16, window, sinks, stale=window == 17)
    K.window_attention(*b.args(), window=window, sinks=sinks, max_query=1)
    plain = b.check(sees)
    b.out.fill_(123.0)
    K.window_attention(*b.args(), window=window, sinks=sinks, max_query=1, workspace=window_ws(b, heads, kv, window, sinks, device, 1))
    split = b.check(sees)
    assert np.abs(plain - split).max() < 0.05


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("heads,kv", [(16, 8), (3, 1), (4, 4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (9, 2), (64, 16), (250, 70)])
def test_window_runs_of_several_tokens(rng, device, f16, heads, kv, window, sinks):
    """Verify runs and prompt chunks, sequences without tokens between them."""
    cached, new = [0, 5, 200, 16, 0, 90, 333], [5, 0, 8, 1, 3, 0, 2]
    for scale in (1, 13):
        b, sees = window_batch(rng, device, cached, np.array(new) * scale, heads, kv, f16, window, sinks)
        ws = window_ws(b, heads, kv, window, sinks, device)
        for workspace, hint in ((None, None), (ws, None), (ws, 1), (None, 1), (None, 10 ** 6)):
            b.out.fill_(123.0)  # a hint below the longest run is slower, not wrong
            K.window_attention(*b.args(), window=window, sinks=sinks, max_query=hint, workspace=workspace)
            b.check(sees)


@pytest.mark.parametrize("cached,new,window,sinks", [(0, 130, 1000, 0), (0, 300, 64, 4), (500, 129, 128, 16), (1000, 257, 300, 1),
                                                     (3, 64, 1, 0), (77, 65, 50, 200), (2048, 128, 2 ** 31 - 1, 0)])
@pytest.mark.parametrize("heads,kv", [(16, 8), (4, 1)])
def test_window_prompt_chunks(rng, device, heads, kv, cached, new, window, sinks):
    b, sees = window_batch(rng, device, [cached], [new], heads, kv, True, window, sinks)
    K.window_attention(*b.args(), window=window, sinks=sinks)
    b.check(sees)
    b.out.fill_(123.0)
    K.window_attention(*b.args(), window=window, sinks=sinks, workspace=window_ws(b, heads, kv, window, sinks, device))
    b.check(sees)


def test_window_long_context_splits_over_several_id_registers(rng, device):
    """A walk of more than 64 pages per split, and splits of a 5000-token window behind freed pages."""
    for f16 in (True, False):
        b, sees = window_batch(rng, device, [6000, 2500], [1, 2], 2, 1, f16, 5000, 20)
        K.window_attention(*b.args(), window=5000, sinks=20, max_query=2)
        b.check(sees)
        b.out.fill_(123.0)
        K.window_attention(*b.args(), window=5000, sinks=20, max_query=2, workspace=window_ws(b, 2, 1, 5000, 20, device, 2))
        b.check(sees)


def test_window_attention_is_the_paged_attention_when_the_window_covers_the_context(rng, device):
    cached, new, H, KV = [100, 700, 33], [1, 1, 1], 16, 8
    b, sees = window_batch(rng, device, cached, new, H, KV, True, 4096, 0, pad_rows=0)
    K.window_attention(*b.args(), window=4096, max_query=1)
    got = b.check(sees)
    b.dev["k"].nan_to_num_(0.0)
    b.dev["v"].nan_to_num_(0.0)
    other = torch.empty_like(b.out)
    ints = K.StepInts(b.pos, np.arange(3), np.where(b.tables < 0, 0, b.tables), b.k.shape[0])
    keep = K.paged_attention(b.dev["q"], b.dev["k"], b.dev["v"], other, ints, n_heads=H, n_kv=KV)
    torch.cuda.synchronize()
    del keep
    assert np.abs(other.double().cpu().numpy() - got).max() < 2e-3 * np.abs(got).max() * 4


def test_window_rows_without_keys_and_positions_outside_the_table(rng, device):
    """A negative position gives zeros; a position past its table sees what its window leaves of the table."""
    b, sees = window_batch(rng, device, [40, 40, 40], [1, 1, 1], 4, 2, True, 30, 0, pad_rows=0)
    W = b.tables.shape[1] * PAGE
    for q_rows in (1, 100):  # the walk and the tile form
        b.pos = np.array([-1, W + 10, W + 40])
        b.dev["pos"] = dint(b.pos, device)
        k, v = (rng.standard_normal(b.k.shape).astype(np.float16) for _ in range(2))
        b.k, b.v, b.dev["k"], b.dev["v"] = k, v, torch.from_numpy(k).to(device), torch.from_numpy(v).to(device)
        b.tables = rng.integers(0, k.shape[0], b.tables.shape)
        b.dev["table"] = dint(b.tables, device)
        b.out.fill_(123.0)
        K.window_attention(*b.args(), window=30, max_query=q_rows)
        b.check(sees)
        assert (b.out[0] == 0).all() and (b.out[2] == 0).all() and (b.out[1] != 0).any()


@pytest.mark.parametrize("window", [1, 7, 2 ** 31 - 2, 2 ** 31 - 1])
def test_window_positions_up_to_the_last_int(rng, device, window):
    """Positions far past the table: the first tokens, and what a window as wide leaves of the table."""
    b, _ = window_batch(rng, device, [100, 100, 100], [1, 1, 1], 4, 2, True, 200, 0, pad_rows=0)
    sees = lambda s, p, j: (j <= p) & ((p - j < window) | (j < 5))  # noqa: E731
    b.pos = np.array([2 ** 31 - 1, 2 ** 31 - 9, 2 ** 31 - 20])
    b.dev["pos"] = dint(b.pos, device)
    k, v = (rng.standard_normal(b.k.shape).astype(np.float16) for _ in range(2))
    b.k, b.v, b.dev["k"], b.dev["v"] = k, v, torch.from_numpy(k).to(device), torch.from_numpy(v).to(device)
    b.tables = rng.integers(0, k.shape[0], b.tables.shape)
    b.dev["table"] = dint(b.tables, device)
    for hint in (1, 100):  # the walk and the tile form
        b.out.fill_(123.0)
        K.window_attention(*b.args(), window=window, sinks=5, max_query=hint)
        b.check(sees)


def test_window_long_tiles_take_page_ids_more_than_once(rng, device):
    """More than 64 blocks in a key group, whose ids are held 64 at a time; the window starts inside a page."""
    b, sees = window_batch(rng, device, [12000], [40], 4, 1, True, 10001, 3)
    K.window_attention(*b.args(), window=10001, sinks=3)
    b.check(sees)


def test_window_blocks_outside_the_pool_read_as_zeros(rng, device):
    b, sees = window_batch(rng, device, [100, 100], [1, 1], 4, 2, True, 200, 0)
    b.tables[0, 2], b.tables[0, 4], b.tables[1, 0], b.tables[1, 6] = b.k.shape[0], -5, 2 ** 31 - 1, -2 ** 31
    b.dev["table"] = dint(b.tables, device)
    b.tables = np.where((b.tables < 0) | (b.tables >= b.k.shape[0]), -1, b.tables)
    for hint in (1, 64):
        b.out.fill_(123.0)
        K.window_attention(*b.args(), window=200, max_query=hint)
        b.check(sees)


@pytest.mark.parametrize("f16,heads,kv,cached,new,window", [
    (True, 4, 2, [100, 31, 40], [1, 1, 1], 64), (True, 8, 1, [100, 31], [3, 1], 64), (False, 4, 2, [100, 31], [3, 1], 64),
    (True, 4, 1, [0, 90], [80, 70], 100), (True, 16, 16, [50] * 10, [200] * 10, 60), (True, 2, 1, [3000], [1], 2500)],
    ids=["decode", "verify", "f32", "tiles", "many tiles", "split"])
def test_window_nan_in_q_stays_in_its_row_and_is_not_hidden(rng, device, f16, heads, kv, cached, new, window):
    b, sees = window_batch(rng, device, cached, np.array(new), heads, kv, f16, window, 3)
    kw = dict(window=window, sinks=3, max_query=max(new), workspace=window_ws(b, heads, kv, window, 3, device, max(new)))
    K.window_attention(*b.args(), **kw)
    b.check(sees)
    _nan_rows(b, heads, lambda: K.window_attention(*b.args(), **kw))


def _nan_rows(b, heads, call):
    clean = b.out.clone()
    rows = [(0, 0), (b.T - 1, heads - 1)]
    for t, h in rows:
        b.dev["q"][t, h, 5 + h] = float("nan")
        clean[t, h] = 0
    b.out.fill_(123.0)
    call()
    for t, h in rows:
        assert torch.isnan(b.out[t, h]).all()
        b.out[t, h] = 0
    assert torch.equal(b.out, clean)


@pytest.mark.parametrize("new", [1, 40])
def test_window_q_inside_wider_rows_and_another_stream(rng, device, new):
    H, KV = 16, 8
    b, sees = window_batch(rng, device, [100, 31], [new, new], H, KV, True, 64, 4)
    wide = torch.full((b.q.shape[0], (H + 2 * KV) * D), float("nan"), dtype=torch.float16, device=device)
    wide[:, KV * D:(KV + H) * D] = b.dev["q"].view(-1, H * D)
    q = wide[:, KV * D:(KV + H) * D].view(-1, H, D)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.window_attention(q, *b.args()[1:], window=64, sinks=4, max_query=new)
    torch.cuda.current_stream().wait_stream(side)
    b.check(sees)
    b.out.fill_(123.0)
    side.wait_stream(torch.cuda.current_stream())
    K.window_attention(q, *b.args()[1:], window=64, sinks=4, max_query=new, stream=side)
    side.synchronize()
    b.check(sees)


def test_attention_over_pages_far_into_a_large_pool(rng, device):
    """Blocks beyond 2^31 elements of the pool, in both forms of both attentions."""
    H, KV, NB = 16, 8, 150_000  # 2.4e9 elements
    far = NB - 1 - np.arange(24).reshape(2, 12)
    k = torch.empty((NB, KV, PAGE, D), dtype=torch.float16, device=device)
    v = torch.empty((NB, KV, PAGE, D), dtype=torch.float16, device=device)
    small = rng.standard_normal((2, 24, KV, PAGE, D)).astype(np.float16)
    k[NB - 24:], v[NB - 24:] = torch.from_numpy(small[0]).to(device), torch.from_numpy(small[1]).to(device)
    for new in (1, 30):
        start, pos = np.array([0, new, 2 * new]), np.concatenate([np.arange(150, 150 + new)] * 2)
        q = rng.standard_normal((2 * new, H, D)).astype(np.float16)
        out = torch.empty((2 * new, H, D), dtype=torch.float16, device=device)
        K.window_attention(torch.from_numpy(q).to(device), k, v, out, dint(start, device), dint(pos, device), dint(far, device),
                           window=100, sinks=8)
        near = far - (NB - 24)
        want, bound = attention_reference(q, small[0], small[1], near, start, pos,
                                          lambda s, p, j: (j <= p) & ((p - j < 100) | (j < 8)), True)
        assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
        far2, near2 = far.copy(), near.copy()
        far2[1, :5], near2[1, :5] = far[0, :5], near[0, :5]
        K.shared_prefix_attention(torch.from_numpy(q).to(device), k, v, out, dint(start, device), dint(pos, device), dint(far2, device),
                                  dint([0, 2], device), dint([80], device),
                                  workspace=K.shared_prefix_workspace(2 * new, 2, 1, n_heads=H, n_kv=KV, device=device))
        want, bound = attention_reference(q, small[0], small[1], near2, start, pos, lambda s, p, j: j <= p, True)
        assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()


def prefix_batch(rng, device, groups, prefix, own, new, heads, kv, f16, **kw):
    """groups: sequences per group; prefix: tokens per group; own, new: per sequence, keys behind the prefix (the new
    tokens among them)."""
    first = np.concatenate([[0], np.cumsum(groups)])
    of = np.repeat(np.arange(len(groups)), groups)
    cached = [prefix[of[s]] + own[s] - new[s] for s in range(len(own))]
    b = Batch(rng, device, cached, new, heads, kv, f16, lambda s, j: np.ones(j.shape, bool),
              shared=lambda s: (int(first[of[s]]), prefix[of[s]]), **kw)
    b.group_start, b.prefix = dint(first, device), dint(prefix, device)
    return b


def causal(s, p, j):
    return j <= p


def prefix_ws(b, heads, kv, device, **hints):
    return K.shared_prefix_workspace(b.q.shape[0], b.cached.size, b.prefix.shape[0], n_heads=heads, n_kv=kv,
                                     dtype=torch.float16 if b.f16 else torch.float32, device=device, **hints)


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("heads,kv", [(16, 8), (6, 2), (2, 2), (12, 1)])
@pytest.mark.parametrize("groups,prefix", [([1], [0]), ([1], [16]), ([3], [37]), ([12], [130]), ([5, 1, 9], [160, 500, 1]),
                                           ([2, 2, 2, 2], [15, 0, 64, 333])])
def test_prefix_decode(rng, device, f16, heads, kv, groups, prefix):
    S = sum(groups)
    own, new = rng.integers(1, 150, S), np.ones(S, int)
    own[0] = 1
    b = prefix_batch(rng, device, groups, prefix, own, new, heads, kv, f16)
    for hints in (dict(), dict(max_query=1, max_group=max(groups), max_prefix=max(prefix), max_own=int(own.max())),
                  dict(max_query=1, max_group=1, max_prefix=0, max_own=1)):
        b.out.fill_(123.0)
        K.shared_prefix_attention(*b.args(), b.group_start, b.prefix, workspace=prefix_ws(b, heads, kv, device, **hints), **hints)
        b.check(causal)


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("heads,kv", [(16, 8), (3, 1)])
def test_prefix_runs_of_several_tokens(rng, device, f16, heads, kv):
    """Verify runs, a prompt's chunk in a group, sequences without tokens, and a group of none."""
    groups, prefix = [4, 3, 1], [200, 47, 16]
    own, new = np.array([5, 60, 9, 2, 17, 3, 100, 40]), np.array([5, 3, 0, 2, 1, 0, 70, 40])
    b = prefix_batch(rng, device, groups, prefix, own, new, heads, kv, f16)
    K.shared_prefix_attention(*b.args(), b.group_start, b.prefix, workspace=prefix_ws(b, heads, kv, device))
    b.check(causal)


def test_prefix_tokens_inside_it_and_sequences_of_no_group(rng, device):
    """Tokens before the prefix's end see the prefix up to themselves; sequences before, between and after the groups
    share nothing."""
    H, KV, NB = 4, 2, 120
    k, v = (rng.standard_normal((NB, KV, PAGE, D)).astype(np.float16) for _ in range(2))
    tables = rng.permutation(NB)[:100].reshape(5, 20)
    tables[2, :6] = tables[1, :6]
    start = np.array([0, 2, 8, 9, 12, 13])
    pos = np.concatenate([[60, 61], np.arange(90, 96), [150], [7, 8, 9], [319]])
    q = rng.standard_normal((13, H, D)).astype(np.float16)
    out = torch.empty((13, H, D), dtype=torch.float16, device=device)
    t = lambda a: torch.from_numpy(a).to(device)  # noqa: E731
    ws = K.shared_prefix_workspace(13, 5, 2, n_heads=H, n_kv=KV, max_prefix=96, max_own=320, device=device)
    for first, lens, hints in (([1, 3, 3], [96, 50], {}), ([1, 3, 4], [96, 400], {}), ([1, 3], [93], dict(max_group=1)),
                               ([1, 1, 3, 3], [5, 96, -4], {})):
        out.fill_(float("nan"))
        K.shared_prefix_attention(t(q), t(k), t(v), out, dint(start, device), dint(pos, device), dint(tables, device),
                                  dint(first, device), dint(lens, device), workspace=ws, max_query=6, **hints)
        want, bound = attention_reference(q, k, v, tables, start, pos, causal, True)
        assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
    # no group at all
    K.shared_prefix_attention(t(q), t(k), t(v), out, dint(start, device), dint(pos, device), dint(tables, device),
                              dint([0], device), dint([], device), workspace=ws, max_query=6)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("f16,heads,kv,groups", [(True, 4, 2, [3, 2]), (True, 16, 1, [9, 4]), (False, 4, 2, [3, 2])],
                         ids=["walks", "tiles", "f32"])
def test_prefix_nan_in_q_stays_in_its_row_and_is_not_hidden(rng, device, f16, heads, kv, groups):
    n = sum(groups)
    b = prefix_batch(rng, device, groups, [333, 90], rng.integers(1, 70, n), np.ones(n, int), heads, kv, f16)
    kw = dict(max_query=1, max_group=max(groups), max_prefix=333, max_own=70)
    ws = prefix_ws(b, heads, kv, device, **kw)
    call = lambda: K.shared_prefix_attention(*b.args(), b.group_start, b.prefix, workspace=ws, **kw)  # noqa: E731
    call()
    b.check(causal)
    _nan_rows(b, heads, call)


def test_prefix_many_groups(rng, device):
    """More groups than a wave has lanes, so a sequence's group is found in two steps."""
    groups = rng.integers(1, 3, 150).tolist()
    S = sum(groups)
    prefix = rng.integers(0, 40, 150).tolist()
    own = rng.integers(1, 30, S)
    b = prefix_batch(rng, device, groups, prefix, own, np.ones(S, int), 4, 2, True)
    K.shared_prefix_attention(*b.args(), b.group_start, b.prefix, workspace=prefix_ws(b, 4, 2, device, max_query=1), max_query=1)
    b.check(causal)


def test_prefix_long_one_in_many_splits(rng, device):
    for heads, kv, n in ((16, 8, 9), (2, 2, 3), (64, 8, 20)):
        b = prefix_batch(rng, device, [n], [2000], rng.integers(1, 40, n), np.ones(n, int), heads, kv, True)
        hints = dict(max_query=1, max_group=n, max_prefix=2000, max_own=40)
        K.shared_prefix_attention(*b.args(), b.group_start, b.prefix, workspace=prefix_ws(b, heads, kv, device, **hints), **hints)
        b.check(causal)


def test_prefix_and_own_keys_of_thousands_of_tokens_unsplit(rng, device):
    """A tile's and a walk's page ids taken more than once, where the workspace allows no splits."""
    own = np.concatenate([[9000, 4200], rng.integers(1, 40, 10)])
    b = prefix_batch(rng, device, [12], [9000], own, np.ones(12, int), 4, 2, True)
    least = torch.empty(2 * b.q.shape[0] * 4 * 130 * 4, dtype=torch.uint8, device=device)
    K.shared_prefix_attention(*b.args(), b.group_start, b.prefix, workspace=least, max_query=1, max_group=12)
    b.check(causal)


def test_small_workspaces(rng, device):
    """Fewer splits where the workspace has room for fewer; an error where not even two partials fit."""
    b = prefix_batch(rng, device, [6], [700], rng.integers(1, 40, 6), np.ones(6, int), 16, 8, True)
    least = 2 * b.q.shape[0] * 16 * 130 * 4
    for n in (least, 3 * least):
        b.out.fill_(123.0)
        K.shared_prefix_attention(*b.args(), b.group_start, b.prefix, workspace=torch.empty(n, dtype=torch.uint8, device=device))
        b.check(causal)
    for ws in (None, torch.empty(least - 1, dtype=torch.uint8, device=device)):
        with pytest.raises(EmberError, match="workspace"):
            K.shared_prefix_attention(*b.args(), b.group_start, b.prefix, workspace=ws)
    w, sees = window_batch(rng, device, [900], [1], 16, 8, True, 800, 4)
    K.window_attention(*w.args(), window=800, sinks=4, max_query=1, workspace=torch.empty(5 * 16 * 130 * 4 * 4, dtype=torch.uint8, device=device))
    w.check(sees)


def test_window_workspace_of_a_large_batch_splits_small_ones_as_their_own_does(rng, device):
    b, sees = window_batch(rng, device, [4000], [1], 16, 8, True, 3900, 4, pad_rows=0)
    outs = []
    for S in (1, 64):
        ws = K.window_workspace(S, S, n_heads=16, n_kv=8, window=3900, sinks=4, max_query=1, device=device)
        b.out.fill_(123.0)
        K.window_attention(*b.args(), window=3900, sinks=4, max_query=1, workspace=ws)
        b.check(sees)
        outs.append(b.out.clone())
    assert torch.equal(*outs)


def test_attention_python_refusals(rng, device):
    b, _ = window_batch(rng, device, [10, 20], [1, 1], 4, 2, True, 8, 0)
    good = b.args()
    call = lambda a, **kw: K.window_attention(*a, **{**dict(window=8), **kw})  # noqa: E731
    swap = lambda at, x: good[:at] + (x,) + good[at + 1:]  # noqa: E731
    for a in (swap(0, good[0].float()), swap(0, good[0].transpose(0, 1)), swap(0, good[0].cpu()), swap(0, good[0][:, :3]),
              swap(0, good[0].bfloat16()), swap(1, good[1][:, :1]), swap(1, good[1].view(-1)), swap(2, good[2].float()),
              swap(3, good[3][:2]), swap(3, good[3].float()), swap(4, good[4].long()), swap(5, good[5][:2]), swap(5, good[5].cpu()),
              swap(6, good[6][:1]), swap(6, good[6].float()), swap(6, good[6][:, ::2])):
        with pytest.raises(EmberError):
            call(a)
    wide = torch.zeros((5, 4 * D + 4), dtype=torch.float16, device=device)[:, :4 * D].view(5, 4, D)  # rows 8 bytes off
    for kw in (dict(window=0), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(workspace=torch.empty(64, dtype=torch.uint8))):
        with pytest.raises(EmberError):
            call(good, **kw)
    with pytest.raises(EmberError):
        call(swap(0, wide))
    with pytest.raises(EmberError):
        K.window_attention(*swap(1, torch.zeros((9, 3, PAGE, D), dtype=torch.float16, device=device))[:2],
                           torch.zeros((9, 3, PAGE, D), dtype=torch.float16, device=device), *good[3:], window=8)  # 4 heads over 3
    gs, pl = dint([0, 2], device), dint([4], device)
    for bad in ((dint([0], device), pl), (gs.long(), pl), (gs, pl.cpu())):
        with pytest.raises(EmberError):
            K.shared_prefix_attention(*good, *bad)


def test_window_sizes_beyond_32_bits_are_refused(rng, device):
    b, _ = window_batch(rng, device, [40], [1], 4, 2, True, 30, 0)
    for window, sinks in ((2 ** 32 + 5, 0), (2 ** 31, 0), (5, 2 ** 32 + 1), (0, 0), (5, -1)):
        with pytest.raises(EmberError):
            K.window_attention(*b.args(), window=window, sinks=sinks)
        with pytest.raises(EmberError):
            K.window_workspace(1, 1, n_heads=4, n_kv=2, window=window, sinks=sinks, device=device)


def test_empty_batches(rng, device):
    b, _ = window_batch(rng, device, [10], [1], 4, 2, True, 8, 0)
    q, k, v, out, start, pos, table = b.args()
    K.window_attention(q[:0], k, v, out[:0], start, pos, table, window=8)
    K.window_attention(q, k, v, out, start[:1], pos, table, window=8)  # no sequences
    K.shared_prefix_attention(q, k, v, out, start[:1], pos, table, dint([0], device), dint([], device))
    torch.cuda.synchronize()
    assert (out == 123.0).all()


# ---- a step as it is used: tables, append, both attentions ----

def _append(t: K.StepTables, qkv, q, k, v, inv, num_blocks, H, KV):
    """The append kernel over a step's device tables, padding rows included."""
    a = _lib.QkvArgs()
    a.qkv, a.q_out, a.k_cache, a.v_cache = qkv.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.inv_freq, a.positions, a.token_seq, a.block_tables = (x.data_ptr() for x in (inv, t.positions, t.token_seq, t.block_tables))
    a.max_blocks, a.T, a.n_heads, a.n_kv, a.head_dim, a.eps = t.max_blocks, t.max_tokens, H, KV, D, 1e-6
    a.num_blocks, a.dtype = num_blocks, _lib.DTYPE_F16
    _lib.check(_lib.lib().ember_hip_kv_append(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), "kv_append")


class Loop:
    """Serving steps of 6 of 8 requests, two of whom share a cached prompt, all on the device: tables, append,
    shared-prefix attention and windowed attention; the lengths and the free list's cursor move on the device."""
    H, KV, S, R, W, CAP = 16, 8, 6, 8, 24, 32

    def __init__(self, device, seed):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.g, self.dev = g, device
        self.blocks = 150
        place = rng.permutation(self.blocks - 1)
        self.spare = self.blocks - 1
        self.cached = np.array([70, 100, 64, 90, 0, 15, 33, 200])
        tables = np.full((self.R, self.W), -1)
        at = 0
        for r, c in enumerate(self.cached):
            n = -(-c // PAGE)
            tables[r, :n] = place[at:at + n]
            at += n
        tables[3, :4] = tables[2, :4]  # requests 2 and 3 share 64 tokens
        self.request = np.array([4, 2, 3, 7, 1, 5])
        self.k, self.v = (torch.randn((self.blocks, self.KV, PAGE, D), generator=g, device=device).half() for _ in range(2))
        self.t = K.StepTables(self.S, self.CAP, self.W, device)
        self.d = dict(tables=dint(tables, device), cached=dint(self.cached, device), new=dint(np.ones(self.S), device),
                      free=dint(place[at:], device), cursor=dint([0], device), request=dint(self.request, device),
                      groups=dint([1, 3], device), prefix=dint([64], device))
        self.inv = torch.from_numpy(K.inv_freq(1e6)).to(device)
        self.qkv = torch.zeros((self.CAP, (self.H + 2 * self.KV) * D), dtype=torch.float16, device=device)
        self.q = torch.zeros((self.CAP, self.H, D), dtype=torch.float16, device=device)
        self.out = torch.zeros_like(self.q), torch.zeros_like(self.q)
        self.ws = (K.window_workspace(self.CAP, self.S, n_heads=self.H, n_kv=self.KV, window=50, sinks=4, max_query=5, device=device),
                   K.shared_prefix_workspace(self.CAP, self.S, 1, n_heads=self.H, n_kv=self.KV, max_query=5, max_group=10,
                                             max_prefix=64, max_own=320, device=device))

    def inputs(self, new):
        self.d["new"].copy_(dint(new, self.dev))
        for o in self.out:
            o.zero_()
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=self.g, device=self.dev).half())

    def step(self):
        d, t = self.d, self.t
        K.step_tables(t, d["tables"], d["cached"], d["new"], d["free"], request=d["request"], free_cursor=d["cursor"], pad_block=self.spare)
        _append(t, self.qkv, self.q, self.k, self.v, self.inv, self.blocks, self.H, self.KV)
        batch = (t.query_start, t.positions, t.block_tables)
        K.shared_prefix_attention(self.q, self.k, self.v, self.out[0], *batch, d["groups"], d["prefix"], max_query=5, max_group=10,
                                  max_prefix=64, max_own=320, workspace=self.ws[1])
        K.window_attention(self.q, self.k, self.v, self.out[1], *batch, window=50, sinks=4, max_query=5, workspace=self.ws[0])
        d["cursor"].copy_(t.totals[1:2])
        d["cached"].index_copy_(0, d["request"].long(), t.context_len)


NEWS = [[1, 1, 1, 1, 1, 1], [5, 1, 3, 0, 1, 2], [1, 0, 5, 5, 4, 1], [2, 2, 2, 2, 2, 2], [1, 1, 1, 1, 1, 1]]


def test_steps_on_the_device_match_the_references(device):
    loop = Loop(device, 5)
    d = loop.d
    for new in NEWS:
        before = {f: d[f].cpu().numpy() for f in ("tables", "cached", "cursor")}
        loop.inputs(new)
        loop.step()
        torch.cuda.synchronize()
        want = step_tables_reference(loop.request, before["cached"], new, before["tables"], d["free"].cpu().numpy(),
                                     int(before["cursor"][0]), loop.CAP, loop.spare)
        for f in FIELDS:
            assert np.array_equal(getattr(loop.t, f).cpu().numpy(), want[f]), f
        assert want["totals"][2] == 0
        assert np.array_equal(d["tables"].cpu().numpy(), want["request_tables"])
        q, k, v = (x.cpu().numpy() for x in (loop.q, loop.k, loop.v))
        T = int(want["totals"][0])
        args = (q[:T], k, v, want["block_tables"][:-1], want["query_start"], want["positions"][:T])
        for got, sees in ((loop.out[0], causal), (loop.out[1], lambda s, p, j: (j <= p) & ((p - j < 50) | (j < 4)))):
            ref, bound = attention_reference(*args, sees, True)
            assert (np.abs(got[:T].double().cpu().numpy() - ref) <= bound).all()
            assert (got[T:] == 0).all()


def test_captured_steps_replay_like_eager_ones(device):
    """One captured step, replayed over steps of other lengths with eager work between the replays, against the same
    steps run eagerly."""
    eager, graphed = Loop(device, 9), Loop(device, 9)
    side = torch.cuda.Stream()
    graphed.inputs(NEWS[0])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up on a twin, so that the graph's own state is untouched
        twin = Loop(device, 11)
        twin.inputs(NEWS[0])
        twin.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.step()
    eager.g.manual_seed(1)
    graphed.g.manual_seed(1)
    for new in NEWS:
        eager.inputs(new)
        eager.step()
        graphed.inputs(new)
        graph.replay()
        twin.step()  # eager work of other buffers between the replays
        torch.cuda.synchronize()
        for f in FIELDS:
            assert torch.equal(getattr(eager.t, f), getattr(graphed.t, f)), f
        # the spare page takes every padding row's K/V in one slot, in any order
        state = lambda loop: (*loop.out, loop.k[:loop.spare], loop.v[:loop.spare], loop.d["cached"], loop.d["tables"])  # noqa: E731
        for a, b in zip(state(eager), state(graphed)):
            assert torch.equal(a, b)


def test_results_do_not_depend_on_other_work_or_repetition(rng, device):
    """The same call again, and beside calls on another stream with a workspace of their own: the same bits."""
    b, _ = window_batch(rng, device, rng.integers(0, 900, 12), np.ones(12, int), 16, 8, True, 500, 4)
    ws = [window_ws(b, 16, 8, 500, 4, device, 1) for _ in range(2)]
    outs = [torch.zeros_like(b.out) for _ in range(6)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, k, v, _, *batch = b.args()
    for i, o in enumerate(outs):
        K.window_attention(q, k, v, o, *batch, window=500, sinks=4, max_query=1, workspace=ws[i % 2], stream=side if i % 2 else None)
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])
