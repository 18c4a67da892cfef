"""The span attentions at their edges: positions and windows at the ends of 32 bits, scores of any size,
long tails of small weights (in the walk and in the tile form), steps of more work-groups
than a launch holds, and padded ones. Step tables of wide and unaligned rows, and the lengths between steps."""
import math

import numpy as np
import pytest
import torch

from ember_amd import _lib
from ember_amd import kernels as K
from span_reference import D, PAGE, attention_reference, step_tables_reference
from test_gpu_span_ops import FIELDS, dint, prefix_batch, prefix_ws, random_tables, window_batch

pytestmark = pytest.mark.gpu

H, KV = 4, 2  # two query heads a kv head: tiles from 9 tokens of one sequence on


def tile_form(b, hint, heads=H, kv=KV):
    """Whether a window call of this batch takes the tile form: more than 16 rows of (token, head of a kv head)."""
    return b.f16 and min(b.q.shape[0], hint) * (heads // kv) > 16


def with_any_pages(b, rng, device):
    """Every table entry a page of finite values, so that any position may be asked for."""
    b.k, b.v = (rng.standard_normal(b.k.shape).astype(b.k.dtype) for _ in range(2))
    b.dev["k"], b.dev["v"] = torch.from_numpy(b.k).to(device), torch.from_numpy(b.v).to(device)
    b.tables = rng.integers(0, b.k.shape[0], b.tables.shape)
    b.dev["table"] = dint(b.tables, device)


def at_positions(b, device, firsts, n):
    """Sequence s at positions firsts[s] .. firsts[s] + n - 1."""
    b.pos = np.concatenate([np.arange(f, f + n) for f in firsts])
    b.dev["pos"] = dint(b.pos, device)


FORMS = pytest.mark.parametrize("n,tiles", [(1, False), (6, False), (10, True), (70, True)])


@FORMS
@pytest.mark.parametrize("window,sinks", [(1, 5), (7, 5), (100, 16), (2 ** 31 - 2, 5), (1, 0), (3000, 100)])
def test_window_positions_up_to_the_last_int_in_both_forms(rng, device, n, tiles, window, sinks):
    """Positions at the end of 32 bits see the first tokens, and nothing where the table has none."""
    b, _ = window_batch(rng, device, [100] * 3, [n] * 3, H, KV, True, 200, 0, pad_rows=0)
    with_any_pages(b, rng, device)
    at_positions(b, device, [2 ** 31 - n, 2 ** 31 - 16 - n, 2 ** 31 - 70 - n], n)
    assert tile_form(b, n) == tiles
    K.window_attention(*b.args(), window=window, sinks=sinks, max_query=n)
    b.check(lambda s, p, j: (j <= p) & ((p - j < window) | (j < sinks)))


@FORMS
def test_window_positions_around_the_table_in_both_forms(rng, device, n, tiles):
    """Negative positions give zeros; positions past the table see what their windows leave of it."""
    b, _ = window_batch(rng, device, [40] * 4, [n] * 4, H, KV, True, 30, 0, pad_rows=0)
    W = b.tables.shape[1] * PAGE
    with_any_pages(b, rng, device)
    at_positions(b, device, [-n, W + 10, W + 40, -n // 2], n)
    assert tile_form(b, n) == tiles
    for sinks in (0, 4):
        b.out.fill_(123.0)
        K.window_attention(*b.args(), window=30, sinks=sinks, max_query=n)
        b.check(lambda s, p, j: (j <= p) & ((p - j < 30) | (j < sinks)))
        assert (b.out[:n] == 0).all()


@FORMS
def test_window_page_ids_outside_the_pool_in_both_forms(rng, device, n, tiles):
    b, sees = window_batch(rng, device, [100, 100], [n, n], H, KV, True, 200, 0)
    b.tables[0, 2], b.tables[0, 4], b.tables[1, 0], b.tables[1, 6] = b.k.shape[0], -5, 2 ** 31 - 1, -2 ** 31
    b.dev["table"] = dint(b.tables, device)
    b.tables = np.where((b.tables < 0) | (b.tables >= b.k.shape[0]), -1, b.tables)
    assert tile_form(b, n) == tiles
    K.window_attention(*b.args(), window=200, max_query=n)
    b.check(sees)


@FORMS
@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
def test_window_of_every_position_but_the_first(rng, device, n, tiles, f16):
    """Window 2^31 - 1: only a token at position 2^31 - 1 is too far from key 0."""
    b, _ = window_batch(rng, device, [100] * 2, [n] * 2, H, KV, f16, 200, 0, pad_rows=0)
    with_any_pages(b, rng, device)
    b.tables[:, 1:] = -1  # key 0's page is what shows
    b.dev["table"] = dint(b.tables, device)
    at_positions(b, device, [2 ** 31 - n, 2 ** 31 - 1 - n], n)
    assert tile_form(b, n) == (tiles and f16)
    K.window_attention(*b.args(), window=2 ** 31 - 1, max_query=n)
    b.check(lambda s, p, j: p - j < 2 ** 31 - 1)


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("n", [1, 12])
def test_prefix_calls_at_the_last_position_see_the_whole_table(rng, device, f16, n):
    """Causal rows have no window: a token at position 2^31 - 1 sees key 0, in a group and in none."""
    b, _ = window_batch(rng, device, [100] * 3, [n] * 3, H, KV, f16, 200, 0, pad_rows=0)
    with_any_pages(b, rng, device)
    b.tables[1, :1] = b.tables[0, :1]
    b.dev["table"] = dint(b.tables, device)
    at_positions(b, device, [2 ** 31 - n] * 3, n)
    for group in ([0, 2], [0, 1]):  # sequences 2, and 1 and 2, are in none
        hints = dict(max_query=n, max_group=2 * n)
        ws = K.shared_prefix_workspace(3 * n, 3, 1, n_heads=H, n_kv=KV, dtype=b.out.dtype, device=device, **hints)
        b.out.fill_(123.0)
        K.shared_prefix_attention(*b.args(), dint(group, device), dint([16], device), workspace=ws, **hints)
        b.check(lambda s, p, j: j <= p)


def largest_score_takes_all(b, sees):
    """Scores so large that the top one's weight is 1 (their gaps exceed what f32 sums lose): its value is the output.
    The only rounding is that of weights and sums, each exact here, and of the output: half a step."""
    torch.cuda.synchronize()
    got = b.out.double().cpu().numpy()
    group = b.q.shape[1] // b.k.shape[1]
    for s in range(len(b.start) - 1):
        for t in range(b.start[s], b.start[s + 1]):
            j = np.arange(b.pos[t] + 1)
            j = j[sees(s, b.pos[t], j)]
            for h in range(b.q.shape[1]):
                k, v = (x[b.tables[s, j // PAGE], h // group, j % PAGE].astype(np.float64) for x in (b.k, b.v))
                e = k @ b.q[t, h].astype(np.float64)
                lost = 130 * 2.0 ** -24 * (np.abs(k) @ np.abs(b.q[t, h].astype(np.float64))).max()
                top = np.sort(e)[::-1]
                if len(e) > 1 and (top[0] - top[1]) * D ** -0.5 < 200 + 2 * lost:
                    continue  # too near a tie for f32
                want = v[e.argmax()]
                step = 2.0 ** -11 if b.f16 else 2.0 ** -21
                assert (np.abs(got[t, h] - want) <= step * np.abs(want)).all(), (t, h, got[t, h][:4], want[:4])


def large(b, device, size, rng):
    """q and keys of this size, random signs and mantissas."""
    for name, x in (("q", b.q), ("k", b.k)):
        x[...] = (size * rng.uniform(0.3, 1, x.shape) * rng.choice([-1, 1], x.shape)).astype(x.dtype)
        b.dev[name] = torch.from_numpy(x).to(device)


@pytest.mark.parametrize("f16,size", [(True, 3e4), (True, 500.0), (False, 1e5), (False, 3e17)])
@pytest.mark.parametrize("n", [1, 6, 12, 70])
@pytest.mark.parametrize("window,sinks", [(1, 0), (50, 0), (400, 3)])
def test_window_scores_of_any_size(rng, device, f16, size, n, window, sinks):
    """Scores of 1e4 to 1e36, positive and negative: weights and sums stay finite, and no row turns into zeros."""
    b, sees = window_batch(rng, device, [0, 300, 40], [n] * 3, H, KV, f16, 10 ** 6, 0)
    large(b, device, size, rng)
    for ws in (None, K.window_workspace(b.q.shape[0], 3, n_heads=H, n_kv=KV, window=window, sinks=sinks, max_query=n,
                                        dtype=b.out.dtype, device=device)):
        b.out.fill_(123.0)
        K.window_attention(*b.args(), window=window, sinks=sinks, max_query=n, workspace=ws)
        largest_score_takes_all(b, lambda s, p, j: (j <= p) & ((p - j < window) | (j < sinks)))


@pytest.mark.parametrize("f16,size", [(True, 3e4), (False, 1e5), (False, 3e17)])
@pytest.mark.parametrize("groups,prefix", [([3, 1], [37, 1]), ([12], [333])])
def test_prefix_scores_of_any_size(rng, device, f16, size, groups, prefix):
    """The same before and behind a shared prefix, whose partials are merged."""
    S = sum(groups)
    b = prefix_batch(rng, device, groups, prefix, rng.integers(1, 90, S), np.ones(S, int), H, KV, f16)
    first = np.concatenate([[0], np.cumsum(groups)])
    large(b, device, size, rng)
    for g, n in enumerate(prefix):  # a partly shared page's copies hold the same keys again
        for s in range(first[g] + 1, first[g + 1]):
            if n % PAGE:
                a, c = b.tables[first[g], n // PAGE], b.tables[s, n // PAGE]
                b.k[c, :, :n % PAGE] = b.k[a, :, :n % PAGE]
    b.dev["k"] = torch.from_numpy(b.k).to(device)
    hints = dict(max_query=1, max_group=max(groups), max_prefix=max(prefix), max_own=90)
    K.shared_prefix_attention(*b.args(), b.group_start, b.prefix, workspace=prefix_ws(b, H, KV, device, **hints), **hints)
    largest_score_takes_all(b, lambda s, p, j: j <= p)


def tail_batch(rng, device, n, keys, depth):
    """n tokens of one sequence behind `keys` keys: key 0 has score 0 and value 0, all others score -depth (base 2, with
    scale ln 2) and value 1: the output is x / (1 + x), x = (keys seen - 1) 2^-depth."""
    b, _ = window_batch(rng, device, [keys], [n], H, KV, True, 10 ** 6, 0)
    b.q[...], b.k[...], b.v[...] = 0, 0, 1
    b.q[..., 0], b.k[..., 0] = 1, -depth
    b.k[b.tables[0, 0], :, 0, 0], b.v[b.tables[0, 0], :, 0] = 0, 0
    for name in "qkv":
        b.dev[name] = torch.from_numpy(getattr(b, name)).to(device)
    return b


def check_tail(b, depth):
    """A weight is rounded by 2^-11 of itself, or by 2^-32 of the largest where f16 ends; exponents (error 2^-22 of
    depth + 2^7, in f32) and sums of up to 2^14 terms in f32 (2^-10 of x at the very most); the output by half a step."""
    torch.cuda.synchronize()
    got = b.out[:b.T].double().cpu().numpy()
    seen = b.pos.astype(np.float64)  # keys 1 .. position
    x = seen * 2.0 ** -depth
    want = (x / (1 + x))[:, None, None]
    tol = want * (2.0 ** -11 + 2.0 ** -11 + (depth + 128) * 2.0 ** -22 + 2.0 ** -10) + seen[:, None, None] * 2.0 ** -32 + 2.0 ** -25
    assert (np.abs(got - want) <= tol).all(), (got.min(), got.max(), want.min())


@pytest.mark.parametrize("n", [1, 6, 12, 70])
@pytest.mark.parametrize("depth", [10, 17, 23, 25, 26])
def test_window_long_tails_of_small_weights_count(rng, device, n, depth):
    """8000 keys of 2^-23 to 2^-26 of the largest weight: less than f16 holds of 1, and up to a thousandth of the row."""
    b = tail_batch(rng, device, n, 8000, depth)
    for ws in (None, K.window_workspace(b.q.shape[0], 1, n_heads=H, n_kv=KV, window=10 ** 6, max_query=n, device=device)):
        b.out.fill_(123.0)
        K.window_attention(*b.args(), window=10 ** 6, max_query=n, scale=math.log(2.0), workspace=ws)
        check_tail(b, depth)


@pytest.mark.parametrize("n", [1, 12])
@pytest.mark.parametrize("prefix", [16, 6016])
def test_prefix_long_tails_of_small_weights_count(rng, device, n, prefix):
    b = tail_batch(rng, device, n, 8000, 25)
    hints = dict(max_query=n, max_group=n, max_prefix=prefix, max_own=8100 - prefix)
    ws = K.shared_prefix_workspace(b.q.shape[0], 1, 1, n_heads=H, n_kv=KV, device=device, **hints)
    K.shared_prefix_attention(*b.args(), dint([0, 1], device), dint([prefix], device), scale=math.log(2.0), workspace=ws, **hints)
    check_tail(b, 25)


def pages_and_tables(rng, device, S, W, dt, blocks=300):
    k, v = (rng.standard_normal((blocks, 8, PAGE, D)).astype(dt) for _ in range(2))
    return k, v, torch.from_numpy(k).to(device), torch.from_numpy(v).to(device), rng.integers(0, blocks, (S, W))


def test_prefix_4096_decodes_without_hints(rng, device):
    """max_query is all 4096 tokens then: 512 row tiles for each of 4096 sequences and 8 kv heads, 2^32 threads if each
    had a work-group."""
    S = 4096
    k, v, dk, dv, tables = pages_and_tables(rng, device, S, 3, np.float16)
    tables[:2000, 0] = tables[0, 0]
    pos = rng.integers(16, 48, S)
    q = rng.standard_normal((S, 16, D)).astype(np.float16)
    out = torch.empty((S, 16, D), dtype=torch.float16, device=device)
    ws = K.shared_prefix_workspace(S, S, 1, n_heads=16, n_kv=8, device=device)
    K.shared_prefix_attention(torch.from_numpy(q).to(device), dk, dv, out, dint(np.arange(S + 1), device), dint(pos, device),
                              dint(tables, device), dint([0, 2000], device), dint([16], device), workspace=ws)
    some = np.unique(np.concatenate([[0, 1, 1999, 2000, S - 1], rng.integers(0, S, 40)]))
    want, bound = attention_reference(q[some], k, v, tables[some], np.arange(len(some) + 1), pos[some], lambda s, p, j: j <= p, True)
    assert (np.abs(out.double().cpu().numpy()[some] - want) <= bound).all()
    assert not torch.isnan(out).any()


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
def test_window_2048_verify_runs_without_hints(rng, device, f16):
    S, n = 2048, 4
    dt = np.float16 if f16 else np.float32
    k, v, dk, dv, tables = pages_and_tables(rng, device, S, 4, dt)
    pos = (rng.integers(0, 60, S)[:, None] + np.arange(n)).reshape(-1)
    q = rng.standard_normal((S * n, 16, D)).astype(dt)
    out = torch.full((S * n, 16, D), float("nan"), dtype=dk.dtype, device=device)
    K.window_attention(torch.from_numpy(q).to(device), dk, dv, out, dint(np.arange(S + 1) * n, device), dint(pos, device),
                       dint(tables, device), window=20, sinks=3)
    some = np.unique(np.concatenate([[0, S - 1], rng.integers(0, S, 12)]))
    rows = (some[:, None] * n + np.arange(n)).reshape(-1)
    want, bound = attention_reference(q[rows], k, v, tables[some], np.arange(len(some) + 1) * n, pos[rows],
                                      lambda s, p, j: (j <= p) & ((p - j < 20) | (j < 3)), f16)
    assert (np.abs(out.double().cpu().numpy()[rows] - want) <= bound).all()
    assert not torch.isnan(out).any()


def test_prefix_partials_of_more_rows_than_one_merge_launch_holds(rng, device):
    """Tokens around row 2^25 and behind row 2^26 of (token, head), the others of no sequence; most of the 105 GB are
    never touched."""
    T = 2 ** 22 + 8
    need = T * 16 * (2 * D * 2 + 2 * (D + 2) * 4)
    if torch.cuda.mem_get_info()[0] < need + (8 << 30):
        pytest.skip(f"needs {need >> 30} GB of free GPU memory")
    k, v, dk, dv, tables = pages_and_tables(rng, device, 3, 4, np.float16)
    tables[1, 0] = tables[0, 0]
    q, out = (torch.empty((T, 16, D), dtype=torch.float16, device=device) for _ in range(2))
    pos = torch.zeros(T, dtype=torch.int32, device=device)
    ws = torch.empty(T * 16 * 2 * (D + 2) * 4, dtype=torch.uint8, device=device)
    for at in (2 ** 21 - 2, T - 5):
        host = rng.standard_normal((5, 16, D)).astype(np.float16)
        where = np.array([40, 41, 20, 50, 51])
        q[at:at + 5], pos[at:at + 5] = torch.from_numpy(host).to(device), dint(where, device)
        out[at - 2:at + 5] = 123.0
        K.shared_prefix_attention(q, dk, dv, out, dint([at, at + 2, at + 3, at + 5], device), pos, dint(tables, device),
                                  dint([0, 2], device), dint([16], device), max_query=2, max_group=3, max_prefix=16, max_own=64,
                                  workspace=ws)
        want, bound = attention_reference(host, k, v, tables, [0, 2, 3, 5], where, lambda s, p, j: j <= p, True)
        assert (np.abs(out[at:at + 5].double().cpu().numpy() - want) <= bound).all()
        assert (out[at - 2:at] == 123.0).all()
    del q, out, ws
    torch.cuda.empty_cache()


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("n", [1, 12])
def test_window_padded_steps_split_as_their_tokens_do(rng, device, f16, n):
    """Rows of padding behind the tokens take no room in the workspace and change no bit."""
    b, sees = window_batch(rng, device, [4000], [n], H, KV, f16, 3900, 4, pad_rows=500)
    q, k, v, out, *batch = b.args()
    outs = []
    for rows in (n, n + 500):
        ws = K.window_workspace(rows, 1, n_heads=H, n_kv=KV, window=3900, sinks=4, max_query=n, dtype=out.dtype, device=device)
        assert ws.nbytes == window_bytes(n, f16)
        out.fill_(123.0)
        K.window_attention(q[:rows], k, v, out[:rows], *batch, window=3900, sinks=4, max_query=n, workspace=ws)
        b.check(sees)
        outs.append(out.clone())
    assert torch.equal(*outs)


def window_bytes(n, f16):
    return K.window_workspace(n, 1, n_heads=H, n_kv=KV, window=3900, sinks=4, max_query=n, device="cpu",
                              dtype=torch.float16 if f16 else torch.float32).nbytes


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("n,hint", [(2, 1), (40, 12), (40, 1)])
def test_window_steps_of_more_tokens_than_named_stay_inside_their_workspace(rng, device, f16, n, hint):
    """One sequence of n tokens, named as `hint`: not split, right, and nothing is written behind the workspace."""
    b, sees = window_batch(rng, device, [4000], [n], H, KV, f16, 3900, 4)
    size = window_bytes(hint, f16)
    room = torch.full((size + 4096,), 77, dtype=torch.uint8, device=device)
    K.window_attention(*b.args(), window=3900, sinks=4, max_query=hint, workspace=room[:size])
    b.check(sees)
    assert (room == 77).all()  # not split: nothing is written at all


# ---- step tables ----

def tables_at(rng, device, W, shift):
    """Step tables whose request rows (or whose own rows) start `shift` entries behind a 16-byte boundary."""
    request, cached, new, tables, free = random_tables(rng, 9, 12, W, W * PAGE - 300, 200)
    want = step_tables_reference(request, cached, new, tables, free, 0, int(new.sum()) + 3, 5)
    flat = torch.full((12 * W + 8,), -77, dtype=torch.int32, device=device)
    rows = flat[shift:shift + 12 * W].view(12, W)
    rows.copy_(dint(tables, device))
    out = K.StepTables(9, int(new.sum()) + 3, W, device)
    K.step_tables(out, rows, dint(cached, device), dint(new, device), dint(free, device), request=dint(request, device), pad_block=5)
    torch.cuda.synchronize()
    for f in FIELDS:
        assert np.array_equal(getattr(out, f).cpu().numpy(), want[f]), f
    assert np.array_equal(rows.cpu().numpy(), want["request_tables"])
    assert (flat[:shift] == -77).all() and (flat[shift + 12 * W:] == -77).all()


@pytest.mark.parametrize("W", [1024, 1028, 2048, 2052, 3100])
def test_step_tables_rows_of_several_segments_four_entries_at_a_time(rng, device, W):
    tables_at(rng, device, W, 0)


@pytest.mark.parametrize("shift", [1, 2, 3, 4])
@pytest.mark.parametrize("W", [24, 1028, 1029])
def test_step_tables_rows_off_a_16_byte_boundary(rng, device, W, shift):
    tables_at(rng, device, W, shift)


def test_step_lengths_survive_an_invalid_step(rng, device):
    """The lengths' update between steps, max(length, context), keeps those of requests that an invalid step left out
    (a negative new_len, a request named twice): their context_len is 0."""
    request = np.array([3, 1, 4, 4, 0])
    cached, new = np.array([40, 17, 5, 64, 90, 33]), np.array([2, -1, 1, 1, 3])
    tables = np.full((6, 8), -1)
    for r, c in enumerate(cached):
        tables[r, :-(-c // PAGE)] = 10 * r + np.arange(-(-c // PAGE))
    out, lengths, rows = K.StepTables(5, 16, 8, device), dint(cached, device), dint(request, device)
    K.step_tables(out, dint(tables, device), lengths, dint(new, device), dint(np.arange(100, 120), device), request=rows)
    at = rows.long()
    lengths.index_copy_(0, at, torch.maximum(lengths[at], out.context_len))
    assert out.context_len.tolist() == [66, 0, 0, 0, 43] and out.totals.tolist()[2] == _lib.STEP_INVALID
    assert lengths.tolist() == [43, 17, 5, 66, 90, 33]


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
def test_window_parts_of_a_step_split_as_steps_of_their_own_do(rng, device, f16):
    """A step's decodes and its chunk in two calls over slices of query_start and the tables, each with the workspace of
    its own tokens: the same bits as when the tokens are a step of their own."""
    cached, new = [4000, 3000, 3500], [1, 1, 40]
    b, sees = window_batch(rng, device, cached, new, H, KV, f16, 3900, 4, pad_rows=20)
    q, k, v, out, start, pos, tables = b.args()
    for s0, s1, n in ((0, 2, 1), (2, 3, 40)):
        a, e = int(b.start[s0]), int(b.start[s1])
        size = dict(n_heads=H, n_kv=KV, window=3900, sinks=4, max_query=n, dtype=out.dtype, device=device)
        ws = K.window_workspace(e - a, s1 - s0, **size)
        assert ws is not None
        ws.fill_(255)  # NaN: only what the call has written may count
        kw = dict(window=3900, sinks=4, max_query=n, workspace=ws)
        K.window_attention(q, k, v, out, start[s0:s1 + 1], pos, tables[s0:s1], **kw)
        alone = torch.empty((e - a, H, D), dtype=out.dtype, device=device)
        K.window_attention(q[a:e], k, v, alone, dint(b.start[s0:s1 + 1] - a, device), pos[a:e], tables[s0:s1], **kw)
        torch.cuda.synchronize()
        assert torch.equal(out[a:e], alone)
    b.check(sees)
