"""The span attentions at their edges: positions and windows at the ends of 32 bits, in the walk and in the tile form."""
import numpy as np
import pytest
import torch

from ember_amd import kernels as K
from span_reference import PAGE
from test_gpu_span_ops import dint, window_batch

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
