"""The 4-bit operators where streams, forms of a launch and scales meet their limits."""
import numpy as np
import pytest
import torch

import four_bit_reference as ref
from ember_amd import _lib
from ember_amd import kernels as K
from four_bit_reference import D, PAGE
from span_reference import attention_reference
from test_gpu_four_bit import attend, batch, check, dint, on

pytestmark = pytest.mark.gpu


def told(b, context, most=None):
    """The batch with tables for `context` keys a sequence, and told that it has that many (and `most` tokens a sequence)."""
    W = context // PAGE
    b["table"] = np.pad(b["table"], ((0, 0), (0, max(0, W - b["W"]))), constant_values=-1)
    b["W"] = b["table"].shape[1]
    b["longest"] = context
    b["most"] = most or b["most"]
    return b


def plan(b, cut=True, pad=0):
    """How the call that attend() makes of the batch is launched."""
    a = _lib.Kv4AttnArgs()
    a.T, a.S, a.max_blocks, a.n_heads, a.n_kv, a.head_dim = b["T"] + pad, len(b["start"]) - 1, b["W"], b["H"], b["KV"], D
    a.dtype, a.max_query, a.max_context = _lib.DTYPE_F16, b["most"], b["longest"]
    if cut:
        a.workspace, a.workspace_bytes = 4096, _lib.lib().ember_hip_kv4_workspace_bytes(a)  # not followed
    out = (_lib.Kv4Launch * 2)()
    return list(out[:_lib.lib().ember_hip_kv4_attn_plan(a, out)])


def keep_busy():
    """Some 20 ms or more of work on the current stream."""
    x = torch.ones(4096, 4096, device="cuda")
    for _ in range(20):
        x = x @ x * 2.0 ** -12
    return x


@pytest.mark.parametrize("handle", [False, True], ids=["object", "handle"])
def test_a_workspace_is_zeroed_in_the_order_of_its_calls_stream(rng, device, handle):
    """The current stream is busy, and the memory that the workspace gets held other bytes: calls on another stream find
    zeros all the same, and all rows of items that are shared out are written."""
    b = batch(rng, device, [(9000, 1), (7000, 1)], 4, 2)
    out = torch.full((2, 4, D), 7.0, dtype=torch.float16, device=device)
    args = (on(b["q"], device), on(b["pages"], device), out, dint(b["start"], device), dint(b["pos"], device), dint(b["table"], device))
    sizes = dict(max_query=1, max_context=b["longest"])
    s = torch.cuda.Stream()
    n = K.kv4_workspace(2, 2, n_heads=4, n_kv=2, device=device, **sizes).numel()
    with torch.cuda.stream(s):
        torch.full((n,), 255, dtype=torch.uint8, device=device)
    torch.cuda.synchronize()
    busy = keep_busy()
    stream = s.cuda_stream if handle else s
    ws = K.kv4_workspace(2, 2, n_heads=4, n_kv=2, device=device, **sizes, stream=stream)
    assert ws.numel() == n
    for _ in range(3):
        K.kv4_attention(*args, **sizes, workspace=ws, stream=stream)
    s.synchronize()
    check(b, out.double().cpu().numpy())
    torch.cuda.synchronize()
    del busy


def test_prepared_tensors_are_not_ones_that_the_current_stream_still_writes(rng, device):
    """Blocks that the current stream has freed, with writes to them still queued there, are not what mx_quantize and
    gemv4_pack return on another stream."""
    x = on(rng.standard_normal((4096, 4096)).astype(np.float32), device)
    codes, scales = K.mx_quantize(x)
    packed = K.gemv4_pack(codes, scales)
    s = torch.cuda.Stream()
    for like, call in ((codes, lambda: K.mx_quantize(x, stream=s)[0]), (scales, lambda: K.mx_quantize(x, stream=s)[1]),
                       (packed, lambda: K.gemv4_pack(codes, scales, stream=s))):
        torch.cuda.synchronize()
        busy = keep_busy()
        freed = torch.empty_like(like)
        at = freed.data_ptr()
        freed.fill_(99)  # runs behind the products
        del freed
        assert torch.empty_like(like).data_ptr() == at  # what an allocation on the current stream would get
        got = call()
        torch.cuda.synchronize()
        assert torch.equal(got, like)
        del busy


# ---- the forms of a launch, told by ember_hip_kv4_attn_plan ----

def mixed_batch(rng, device, H, KV, context=30_000):
    """Many decodes, short runs and a few chunks; sequences of 16 and 17 rows, and without tokens."""
    G = H // KV
    new = [1] * 60 + [5, 90, 0, 17, 130, 16, 1, max(1, 16 // G), 16 // G + 1, max(1, 32 // G), 32 // G + 1]
    seqs = [(int(c), n) for c, n in zip(rng.integers(0, 500, len(new)), new)] + [(3000, 1), (2600, 70)]
    return told(batch(rng, device, seqs, H, KV), context)


@pytest.mark.parametrize("cut", [True, False])
@pytest.mark.parametrize("H,KV", [(2, 2), (4, 2), (16, 8), (8, 1), (32, 2)])
def test_steps_of_decodes_and_chunks_in_two_launches(rng, device, H, KV, cut):
    """Short runs in the walk, dealt or shared out, the others on tiles: with one workspace, and without."""
    b = mixed_batch(rng, device, H, KV)
    both = plan(b, cut, pad=3)
    assert [(x.rows, x.least) for x in both] == [(16, 1), (128, 17)]
    assert (both[1].sharers > 0) == cut and (both[0].dealt or (both[0].sharers > 0) == cut)
    check(b, attend(b, device, cut=cut, pad=3))


def test_steps_in_two_launches_of_decodes_alone(rng, device):
    """A server's fixed hints: the second launch finds no chunks."""
    b = told(batch(rng, device, [(int(c), 1) for c in rng.integers(0, 700, 32)], 16, 8), 32_768, most=512)
    assert len(plan(b)) == 2
    check(b, attend(b, device))


def test_steps_in_two_launches_of_chunks_alone(rng, device):
    """The first launch finds no decodes."""
    b = told(batch(rng, device, [(int(c), n) for c, n in zip(rng.integers(0, 300, 40), [0] * 36 + [20, 130, 9, 64])], 4, 2), 30_000)
    assert len(plan(b)) == 2
    check(b, attend(b, device))


def test_steps_in_two_launches_of_more_sequences_than_one_takes(rng, device):
    new = np.ones(4200, int)
    new[[5, 4095, 4096, 4199]] = 40, 70, 33, 18
    b = told(batch(rng, device, [(int(c), int(n)) for c, n in zip(rng.integers(0, 40, 4200), new)], 1, 1), 512)
    assert len(plan(b)) == 2
    check(b, attend(b, device, pad=1))


def test_steps_in_two_launches_captured_and_replayed(rng, device):
    b = mixed_batch(rng, device, 4, 2)
    assert all(x.sharers > 0 for x in plan(b)) and len(plan(b)) == 2
    out = torch.zeros(b["T"], 4, D, dtype=torch.float16, device=device)
    args = (on(b["q"], device), on(b["pages"], device), out, dint(b["start"], device), dint(b["pos"], device), dint(b["table"], device))
    hints = dict(max_query=b["most"], max_context=b["longest"])
    own, other = (K.kv4_workspace(b["T"], len(b["start"]) - 1, n_heads=4, n_kv=2, device=device, **hints) for _ in range(2))
    K.kv4_attention(*args, **hints, workspace=other)
    check(b, out.double().cpu().numpy())
    eager = out.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        K.kv4_attention(*args, **hints, workspace=own)
    for _ in range(4):
        out.fill_(7.0)
        graph.replay()
        assert torch.equal(out, eager)
        out.fill_(7.0)
        K.kv4_attention(*args, **hints, workspace=other)
        assert torch.equal(out, eager)


HEADS = [(16, 8), (4, 2), (8, 1), (3, 1), (5, 5), (12, 1)]


@pytest.mark.parametrize("H,KV", HEADS)
@pytest.mark.parametrize("kind", ["decodes", "runs", "prompts"])
def test_short_and_long_sequences_shared_out(rng, device, H, KV, kind):
    """The edges of pages and steps where the items' keys are shared out, most of them by few work-groups or by one."""
    seqs = dict(decodes=[(c, 1) for c in (0, 1, 15, 16, 63, 64, 65, 300, 1000)],
                runs=[(0, 5), (14, 3), (61, 6), (200, 1), (399, 2), (777, 4)],
                prompts=[(0, 1), (0, 70), (33, 150), (500, 97), (40, 0), (3, 2)])[kind]
    b = told(batch(rng, device, seqs, H, KV), 40_000)
    assert [x.sharers > 0 for x in plan(b, pad=3)] == [True]
    check(b, attend(b, device, pad=3, strided=kind == "runs"))


@pytest.mark.parametrize("H,KV,new", [(2, 1, 1), (3, 1, 1), (4, 1, 7), (12, 1, 3)])
def test_more_sequences_than_lanes_shared_out(rng, device, H, KV, new):
    """Shares are found by a scan over several loads of lengths: of decodes, of up to 32 rows and of tiles."""
    seqs = [(int(c), int(n)) for c, n in zip(rng.integers(0, 400, 150), rng.integers(0, new + 1, 150))] + [(9000, new), (5000, 1)]
    b = told(batch(rng, device, seqs, H, KV), 200_000)
    form = plan(b)
    assert len(form) == 1 and form[0].sharers > 0 and form[0].rows == (16 if new == 1 else 32 if H == 4 else 128)
    check(b, attend(b, device))


@pytest.mark.parametrize("S,H,KV,most", [(64, 32, 8, 8), (170, 12, 2, 5), (47, 24, 8, 10), (250, 4, 2, 16)])
def test_runs_of_up_to_32_rows_dealt_by_length(rng, device, S, H, KV, most):
    seqs = [(int(c), int(n)) for c, n in zip(rng.choice([0, 16, 33, 150, 500], S), rng.integers(0, most + 1, S))]
    seqs[S // 2], seqs[0] = (2000, most), (7, 0)
    b = told(batch(rng, device, seqs, H, KV), 4096, most=most)
    assert [(x.rows, x.dealt) for x in plan(b, pad=2)] == [(32, 1)]
    check(b, attend(b, device, pad=2))
    check(b, attend(b, device, cut=False))


@pytest.mark.parametrize("cut", [True, False])
@pytest.mark.parametrize("H,KV,forms", [(17, 1, [(32, 1), (128, 33)]), (40, 2, [(32, 1), (128, 33)]), (64, 2, [(32, 1), (128, 33)]), (33, 1, [(128, 1)])])
def test_mixed_steps_of_many_heads_a_kv_head(rng, device, H, KV, forms, cut):
    """A token has more than 16 rows: decodes are walked 32 rows at a time, or are tiles too."""
    b = mixed_batch(rng, device, H, KV)
    assert [(x.rows, x.least) for x in plan(b, cut, pad=3)] == forms
    check(b, attend(b, device, cut=cut, pad=3))


# ---- scales that the quantiser never writes ----

def f16(x):
    """What a value is where it is read: rounded to f16, in float64."""
    with np.errstate(over="ignore"):
        return x.astype(np.float16).astype(np.float64)


LEVELS = np.concatenate([ref.LEVELS, -ref.LEVELS])  # of codes 0 .. 15
FORMS = pytest.mark.parametrize("H", [1, 20, 40], ids=["walk of 16 rows", "walk of 32 rows", "tile"])


def lay_out(k_code, k_scale, v_code, v_scale):
    """Pages [n, PAGE_BYTES] of codes [n, 16, 128] and scale bytes [n, 16, 4]."""
    n = len(k_code)
    v = ref.pack(v_code).reshape(n, 4, 4, 16, 4).swapaxes(2, 3)
    return np.concatenate([ref.pack(k_code).reshape(n, -1), v.reshape(n, -1), k_scale.reshape(n, -1), v_scale.swapaxes(1, 2).reshape(n, -1)], 1)


def attend_pages(device, q, pages, scale):
    """One token of each sequence at position 15 of its own page."""
    S, H, _ = q.shape
    out = torch.zeros(S, H, D, dtype=torch.float16, device=device)
    K.kv4_attention(on(q, device), on(pages, device), out, dint(np.arange(S + 1), device), dint(np.full(S, 15), device),
                    dint(np.arange(S)[:, None], device), max_query=1, max_context=16, scale=scale)
    return out.double().cpu().numpy()


@FORMS
@pytest.mark.parametrize("key", range(4))
def test_values_of_every_finite_scale(rng, device, H, key):
    """V of one key, the others' weights 0: every code at every scale up to the highest that the append writes, at each of
    the four places of a word of scales, whose other bytes are arbitrary."""
    S = 36  # four groups of 32 dims each: 144 scales
    at = 4 * (np.arange(S) % 4) + key
    v_code, k_code = np.zeros((2, S, PAGE, D), np.uint8)
    v_scale, k_scale = rng.integers(0, 255, (2, S, PAGE, 4)).astype(np.uint8)
    s = np.arange(S)
    code = (np.arange(D) + rng.integers(0, 16, (S, 1))).astype(np.uint8) % 16
    byte = ((4 * s[:, None] + np.arange(4)) % 141).astype(np.uint8)
    v_code[s, at], v_scale[s, at] = code, byte
    k_code[s, at], k_scale[s, at] = 7, 127  # 6 in every dim: a score of 768 * 128^-1/2 = 68, the others' 0
    q = np.ones((S, H, D), np.float16)
    got = attend_pages(device, q, lay_out(k_code, k_scale, v_code, v_scale)[:, None], None)
    want = f16(LEVELS[code] * np.repeat(2.0 ** (byte - 127.0), 32, -1))
    assert np.array_equal(got, np.broadcast_to(want[:, None], got.shape))  # the one weight is 2^7 in f16, as is their sum


@FORMS
def test_keys_of_every_finite_scale(rng, device, H):
    """One dim of one key against 15 keys of score 0, in every code and scale; out is that key's weight."""
    byte, code = (x.reshape(-1) for x in np.meshgrid(np.arange(141), [c for c in range(16) if c % 8]))
    for some, scale in ((byte <= 121, 1024.0), (byte > 121, 1.0)):
        b, c = byte[some], code[some]
        S = b.size
        s, at, dim = np.arange(S), rng.integers(0, PAGE, S), rng.integers(0, D, S)
        v_code, k_code = np.zeros((2, S, PAGE, D), np.uint8)
        v_scale, k_scale = rng.integers(0, 255, (2, S, PAGE, 4)).astype(np.uint8)
        k_code[s, at, dim], k_scale[s, at, dim // 32] = c, b
        v_code[s, at], v_scale[s, at] = 2, 127
        k = f16(LEVELS[c] * 2.0 ** (b - 127.0))
        q = rng.standard_normal((S, 1, D)).astype(np.float16)
        q[s, 0, dim] = np.where(k == 0, 1, 3 / np.where(k == 0, 1, k) / scale)  # a score of 3 where k is not 0
        got = attend_pages(device, q.repeat(H, 1), lay_out(k_code, k_scale, v_code, v_scale)[:, None], scale)
        keys, vals = np.zeros((2, S, 1, PAGE, D))
        keys[s, 0, at, dim], vals[s, 0, at] = k, 1
        want, bound = attention_reference(q, keys, vals, s[:, None], np.arange(S + 1), np.full(S, 15), lambda s, p, j: j <= p, True, scale)
        assert (np.abs(got - want) <= bound).all()
        assert (np.abs(want - 1 / 16) > 0.3)[k != 0].all()  # a key that counts is told from one that reads as 0


@pytest.mark.parametrize("M,k", [(1, 128), (40, 1152), (64, 2304), (3, 4224), (200, 4224), (3, 8320)],
                         ids=["rows", "two blocks a wave", "four blocks a wave", "eight blocks a wave", "prompt", "long"])
def test_weights_of_every_scale(rng, device, M, k):
    """Every code at every scale in a product with ones: f16's subnormals, infinities and the NaN scale among them, beside
    arbitrary scales of groups that hold zeros."""
    byte, code = (x.reshape(-1) for x in np.meshgrid(np.arange(256), np.arange(16)))
    N = byte.size
    scales = rng.integers(0, 255, (N, k // 32)).astype(np.uint8)
    codes = np.zeros((N, k), np.uint8)
    n, col = np.arange(N), rng.integers(0, k, N)
    codes[n, col], scales[n, col // 32] = code, byte
    w = K.gemv4_pack(on(ref.pack(codes), device), on(scales, device))
    c = torch.empty(M, N, device=device)
    K.gemv4(torch.ones(M, k, dtype=torch.float16, device=device), w, c, _lib.EPILOGUE_STORE_F32, N=N)
    want = np.where(byte == 255, np.nan, f16(LEVELS[code] * 2.0 ** (byte - 127.0)))
    assert np.array_equal(c.double().cpu().numpy(), np.broadcast_to(want, (M, N)), equal_nan=True)


# ---- positions ----

@pytest.mark.parametrize("shared", [False, True], ids=["an item each", "shared out"])
@pytest.mark.parametrize("n,H,KV,rows", [(1, 4, 2, 16), (6, 4, 1, 32), (70, 4, 2, 128), (1, 40, 1, 128)])
def test_positions_at_the_ends_of_their_range(rng, device, n, H, KV, rows, shared):
    """Negative ones see nothing, those past the table all of it, also at the end of 32 bits; runs that cross both borders."""
    W = 40
    full = batch(rng, device, [(W * PAGE - n, n)] * 7, H, KV, W=W)
    firsts = [-n, -(n // 2), W * PAGE - 1, W * PAGE - n // 2, 2 ** 31 - n, 2 ** 31 - n - 16, -2 ** 31]
    full["pos"] = np.concatenate([f + np.arange(n) for f in firsts])
    if shared:
        told(full, 100_000)
    else:
        full["longest"] = 64
    assert [(x.rows, x.sharers > 0) for x in plan(full)] == [(rows, shared)]
    got = attend(full, device)
    assert (got[full["pos"] < 0] == 0).all()
    check(full, got)


@pytest.mark.parametrize("seed", range(8))
def test_steps_of_any_kind(seed, device):
    """Sequences, heads, hints, strides and missing pages at random."""
    rng = np.random.default_rng(seed)
    KV = int(rng.choice([1, 2, 3, 8]))
    H = KV * int(rng.choice([1, 2, 3, 5, 8, 16, 18, 33][: 5 if KV == 8 else 8]))
    S = int(2 ** rng.uniform(0, 7))
    new = np.where(rng.random(S) < 0.8, 1, (2 ** rng.uniform(0, 7.5, S)).astype(int) - 1)
    seqs = [(int(c), int(m)) for c, m in zip(2 ** rng.uniform(0, 9.5, S) - 1, new)]
    b = batch(rng, device, seqs, H, KV)
    b["table"][rng.random(b["table"].shape) < 0.02] = int(rng.choice([-1, -7, b["pages"].shape[0], 2 ** 31 - 1]))
    missing = (b["table"] < 0) | (b["table"] >= b["pages"].shape[0])
    pad, strided = int(rng.integers(0, 4)), bool(rng.integers(0, 2))
    seen = {**b, "table": np.where(missing, -1, b["table"])}
    for context in (0, 3000, 60_000):
        told(b, max(context, int(rng.integers(1, 1000))), most=int(rng.choice([1, 8, 200])))
        told(seen, b["longest"])
        check(seen, attend(b, device, cut=bool(rng.integers(0, 4)), pad=pad, strided=strided, scale=0.05), 0.05)
