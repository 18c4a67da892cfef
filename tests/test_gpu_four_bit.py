"""A cache and weights in 4 bits on the GPU, against numpy / float64 references.

Slots that no token may see hold bytes that read as NaN, pages that are not needed are -1 in the tables, and rows that
belong to no sequence must keep what they held. The attention's bounds are span_reference's, over what the pages stand
for; the products' are derived beside them.
"""
import numpy as np
import pytest
import torch

import four_bit_reference as ref
from ember_amd import _lib
from ember_amd import kernels as K
from ember_amd._lib import EmberError
from four_bit_reference import D, PAGE, PAGE_BYTES
from span_reference import attention_reference

pytestmark = pytest.mark.gpu


def dint(a, device):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)


def on(a, device):
    return torch.from_numpy(np.ascontiguousarray(a)).to(device)


# ---- quantise ----

@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols,wide", [(1, 32, 0), (3, 96, 5), (70, 4096, 0), (1000, 64, 64), (5, 33 * 32, 1)])
def test_quantize_is_the_definition(rng, device, dtype, rows, cols, wide):
    x = rng.standard_normal((rows, cols + wide)) * 2.0 ** rng.integers(-14, 8, (rows, 1))
    x = on(x, device).to(dtype)
    codes, scales = K.mx_quantize(x[:, :cols])
    code, scale = ref.encode(x[:, :cols].double().cpu().numpy())
    assert np.array_equal(scales.cpu().numpy(), scale)
    assert np.array_equal(codes.cpu().numpy(), ref.pack(code))


def test_quantize_borders_and_extremes(device):
    """Every border between two codes and its neighbours, at every scale; sizes beyond and below the scales."""
    rows = []
    for e in range(-23, 14):
        edge = np.float32([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.0])
        near = np.concatenate([edge, np.nextafter(edge, np.float32(9)), np.nextafter(edge, np.float32(-9)), -edge]).astype(np.float32)
        near[-1] = 7.0  # fixes the group's scale
        rows.append(near * np.float32(2.0 ** e))
        just = near.copy()
        just[-1] = np.nextafter(np.float32(7), np.float32(8))
        rows.append(just * np.float32(2.0 ** e))
    rows += [np.full(32, v, np.float32) for v in (0.0, -0.0, 1e-45, 1e-30, 3e38, -3e38, 65504, 2.0 ** -24)]
    x = np.stack(rows)
    x[-1, 5] = -0.0
    codes, scales = K.mx_quantize(on(x, device))
    code, scale = ref.encode(x)
    assert np.array_equal(scales.cpu().numpy(), scale) and np.array_equal(codes.cpu().numpy(), ref.pack(code))


def test_quantize_nan_and_infinity(device):
    x = torch.ones(3, 64, device=device)
    x[0, 3], x[1, 40], x[2, 63] = float("nan"), float("inf"), float("-inf")
    codes, scales = (t.cpu().numpy() for t in K.mx_quantize(x))
    assert scales.tolist() == [[255, 125], [125, 140], [125, 140]]
    v = ref.decode(ref.unpack(codes), scales)
    assert np.isnan(v[0, :32]).all() and (v[0, 32:] == 1).all() and (v[1, :32] == 1).all()
    assert v[1, 40] == 6 * 2.0 ** 13 and v[2, 63] == -6 * 2.0 ** 13


# ---- append ----

def append_case(rng, device, seqs, H, KV, norm, bias, top=500, W=40):
    """seqs: (cached, new) of each sequence. Returns the call's tensors and the host's view of them."""
    T = sum(n for _, n in seqs)
    blocks = len(seqs) * W + 3
    table = rng.permutation(blocks)[: len(seqs) * W].reshape(len(seqs), W)
    pos = np.concatenate([c + np.arange(n) for c, n in seqs]) if T else np.zeros(0, int)
    seq = np.repeat(np.arange(len(seqs)), [n for _, n in seqs])
    qkv = (2 * rng.standard_normal((T, (H + 2 * KV) * D))).astype(np.float16)
    f32 = lambda *s: on(rng.standard_normal(s).astype(np.float32), device)  # noqa: E731
    t = dict(qkv=on(qkv, device), pos=dint(pos, device), seq=dint(seq, device), table=dint(table, device),
             pool=torch.full((blocks, KV, PAGE_BYTES), 77, dtype=torch.uint8, device=device),
             q_out=torch.zeros(T, H, D, dtype=torch.float16, device=device),
             kw=dict(n_heads=H, n_kv=KV, inv_freq_dev=on(K.inv_freq(1e6), device), q_norm=f32(D) if norm else None,
                     k_norm=f32(D) if norm else None, bias=f32((H + 2 * KV) * D) if bias else None))
    return t, table, pos, seq


def f32_pages(t, table, pos, seq, H, KV, device):
    """What the f32 cache's append makes of the same inputs: q, and K and V of each token in float64."""
    blocks = t["pool"].shape[0]
    ints = K.StepInts(pos, seq, table, blocks)
    kp, vp = torch.zeros(2, blocks, KV, PAGE, D, device=device)
    q = torch.zeros(len(pos), H, D, device=device)
    kw = dict(t["kw"])
    K.qk_norm_rope_store(t["qkv"].float(), q, kp, vp, ints, n_heads=kw.pop("n_heads"), n_kv=kw.pop("n_kv"), **kw)
    blk, slot = table[seq, pos // PAGE], pos % PAGE
    return q, kp.cpu().numpy()[blk, :, slot], vp.cpu().numpy()[blk, :, slot]


SEQS = [[(0, 1)], [(3, 1), (15, 1), (16, 1), (500, 1)], [(0, 37), (5, 1), (30, 130)], [(7, 2)] * 33]


@pytest.mark.parametrize("H,KV", [(16, 8), (4, 2), (5, 5), (8, 1), (12, 4)])
@pytest.mark.parametrize("norm,bias", [(True, False), (False, True)])
@pytest.mark.parametrize("seqs", SEQS, ids=["one", "edges", "ragged", "many"])
def test_append_is_the_f32_append_in_four_bits(rng, device, seqs, H, KV, norm, bias):
    """Pages byte for byte what the f32 append's K and V encode to, nothing else written; q bit for bit the f16 append's."""
    t, table, pos, seq = append_case(rng, device, seqs, H, KV, norm, bias)
    T = len(pos)
    k_out, v_out = torch.zeros(2, T, KV, D, dtype=torch.float16, device=device)
    K.kv4_append(t["qkv"], t["q_out"], t["pool"], t["pos"], t["seq"], t["table"], **t["kw"], k_out=k_out, v_out=v_out)
    q32, k, v = f32_pages(t, table, pos, seq, H, KV, device)
    assert torch.equal(t["q_out"], q32.half())
    want = np.full(t["pool"].shape, 77, np.uint8)
    for i in range(T):
        for h in range(KV):
            ref.write_slot(want[table[seq[i], pos[i] // PAGE], h], pos[i] % PAGE, k[i, h], v[i, h])
    assert np.array_equal(t["pool"].cpu().numpy(), want)
    assert np.array_equal(k_out.cpu().numpy(), ref.decode(*ref.encode(k))) and np.array_equal(v_out.cpu().numpy(), ref.decode(*ref.encode(v)))
    again = t["pool"].clone()  # without the values' outputs: the same pages
    again.fill_(77)
    K.kv4_append(t["qkv"], t["q_out"], again, t["pos"], t["seq"], t["table"], **t["kw"])
    assert torch.equal(again, t["pool"])


def test_append_far_positions(rng, device):
    t, table, pos, seq = append_case(rng, device, [(131000, 3), (1 << 20, 2)], 4, 2, True, False, W=(1 << 16) + 1)
    K.kv4_append(t["qkv"], t["q_out"], t["pool"], t["pos"], t["seq"], t["table"], **t["kw"])
    q32, k, v = f32_pages(t, table, pos, seq, 4, 2, device)
    assert torch.equal(t["q_out"], q32.half())
    got_k, got_v = ref.read_pages(t["pool"][t["table"].long()[t["seq"].long(), t["pos"].long() // PAGE]].cpu().numpy())
    at = np.arange(len(pos)), slice(None), pos % PAGE
    assert np.array_equal(got_k[at], ref.decode(*ref.encode(k))) and np.array_equal(got_v[at], ref.decode(*ref.encode(v)))


def test_append_writes_nothing_where_there_is_no_slot(rng, device):
    t, table, pos, seq = append_case(rng, device, [(0, 8)], 4, 2, True, False, W=3)
    bad_pos = pos.copy()
    bad_pos[:3] = -1, 3 * PAGE, 2 ** 31 - 1
    bad_seq = seq.copy()
    bad_seq[3:6] = -1, 1, 2 ** 31 - 1
    table = table.copy()
    table[0, 0] = t["pool"].shape[0]  # outside the pool
    for tab in (table, np.where(np.arange(3) == 0, -5, table)):
        K.kv4_append(t["qkv"], t["q_out"], t["pool"], dint(bad_pos, device), dint(bad_seq, device), dint(tab, device), **t["kw"])
        assert (t["pool"] == 77).all()
    assert t["q_out"].abs().sum(-1).min() > 0


def test_append_clamps_what_is_not_finite(rng, device):
    t, *_ = append_case(rng, device, [(0, 3)], 2, 1, False, False)
    x = t["qkv"].view(3, 4, D)
    x[:, 3] = 1.0
    x[0, 3, 5], x[1, 3, 40], x[2, 3, 127] = float("inf"), float("-inf"), float("nan")
    v_out, k_out = torch.zeros(2, 3, 1, D, dtype=torch.float16, device=device)
    K.kv4_append(t["qkv"], t["q_out"], t["pool"], t["pos"], t["seq"], t["table"], **t["kw"], k_out=k_out, v_out=v_out)
    assert v_out[0, 0, 5] == 49152 and v_out[1, 0, 40] == -49152 and v_out[2, 0, 127] == -49152
    assert (v_out[0, 0, 32:] == 1).all() and v_out.isfinite().all()


# ---- attention ----

def batch(rng, device, seqs, H, KV, W=None, spread=1.0, garbage=255):
    """seqs: (cached, new). Pages of every sequence hold its keys; other slots of them read as NaN (scale 255)."""
    n = [(c, m) for c, m in seqs]
    need = [-(-(c + m) // PAGE) for c, m in n]
    W = W or max(need + [1]) + 1
    blocks = sum(need) + 3
    place = rng.permutation(blocks)
    table = np.full((len(n), W), -1)
    used = 0
    for s, k in enumerate(need):
        table[s, :k] = place[used:used + k]
        used += k
    k = spread * rng.standard_normal((blocks, KV, PAGE, D)) * np.exp(0.5 * rng.standard_normal(D))
    v = rng.standard_normal((blocks, KV, PAGE, D))
    pages = ref.to_pages(k, v)
    live = np.zeros((blocks, PAGE), bool)
    for s, (c, m) in enumerate(n):
        for j in range(c + m):
            live[table[s, j // PAGE], j % PAGE] = True
    dead = ~live
    for b, sl in zip(*np.nonzero(dead)):
        pages[b, :, 2048 + 4 * sl:2052 + 4 * sl] = garbage
        pages[b, :, 2112 + sl::16] = garbage
    start = np.concatenate([[0], np.cumsum([m for _, m in n])]).astype(int)
    pos = np.concatenate([c + np.arange(m) for c, m in n]) if n else np.zeros(0)
    T = int(start[-1])
    q = (rng.standard_normal((T, H, D)) * 1.5).astype(np.float16)
    return dict(q=q, pages=pages, table=table, start=start, pos=pos.astype(int), T=T, H=H, KV=KV, W=W,
                most=max([m for _, m in n] + [1]), longest=max([c + m for c, m in n] + [1]))


def attend(b, device, cut=True, scale=None, hints=True, pad=0, strided=False):
    """The call, with `pad` rows behind the last sequence that must stay as they are."""
    T, H, KV = b["T"] + pad, b["H"], b["KV"]
    q = torch.zeros(T, H + 3 if strided else H, D, dtype=torch.float16, device=device)
    q[: b["T"], :H] = on(b["q"], device)
    q = q[:, :H] if strided else q
    out = torch.full((T, H, D), 7.0, dtype=torch.float16, device=device)
    S = len(b["start"]) - 1
    named = dict(max_query=b["most"], max_context=b["longest"]) if hints else {}
    sizes = dict(named) if hints else dict(max_blocks=b["W"])
    ws = K.kv4_workspace(T, S, n_heads=H, n_kv=KV, device=device, **sizes) if cut else None
    pos = np.concatenate([b["pos"], np.full(pad, 3)])
    args = (q, on(b["pages"], device), out, dint(b["start"], device), dint(pos, device), dint(b["table"], device))
    K.kv4_attention(*args, scale=scale, workspace=ws, **named)
    first = out.clone()
    for _ in range(2):  # the workspace is left as it was found, and the bits do not depend on who merges
        out.fill_(7.0)
        K.kv4_attention(*args, scale=scale, workspace=ws, **named)
        assert torch.equal(out.nan_to_num(9), first.nan_to_num(9))
    assert (out[b["T"]:] == 7).all()
    return out[: b["T"]].double().cpu().numpy()


def check(b, got, scale=None):
    k, v = ref.read_pages(b["pages"])
    want, bound = attention_reference(b["q"], k, v, b["table"], b["start"], b["pos"], lambda s, p, j: j <= p, True, scale)
    far = np.abs(got - want)
    assert (far <= bound).all(), (far - bound).max()


HEADS = [(16, 8), (4, 2), (8, 1), (3, 1), (5, 5), (12, 1)]


@pytest.mark.parametrize("cut", [True, False])
@pytest.mark.parametrize("H,KV", HEADS)
def test_attention_of_decodes(rng, device, H, KV, cut):
    b = batch(rng, device, [(c, 1) for c in (0, 1, 15, 16, 63, 64, 65, 300, 1000)], H, KV)
    check(b, attend(b, device, cut, pad=3))


@pytest.mark.parametrize("cut", [True, False])
@pytest.mark.parametrize("H,KV", HEADS)
def test_attention_of_verify_runs(rng, device, H, KV, cut):
    b = batch(rng, device, [(0, 5), (14, 3), (61, 6), (200, 1), (399, 2), (777, 4)], H, KV)
    check(b, attend(b, device, cut, pad=2, strided=True))


@pytest.mark.parametrize("cut", [True, False])
@pytest.mark.parametrize("H,KV", [(16, 8), (4, 2), (8, 1), (3, 1)])
def test_attention_of_prompts(rng, device, H, KV, cut):
    b = batch(rng, device, [(0, 1), (0, 70), (33, 150), (500, 97), (40, 0), (3, 2)], H, KV)
    check(b, attend(b, device, cut, pad=5))


@pytest.mark.parametrize("context", [511, 512, 1023, 4097, 20000])
def test_attention_of_long_contexts(rng, device, context):
    b = batch(rng, device, [(context, 1), (context // 3, 1)], 4, 2)
    check(b, attend(b, device))


@pytest.mark.parametrize("H,KV", [(4, 2), (8, 1), (3, 1)])
def test_attention_of_long_contexts_shared_out(rng, device, H, KV):
    """Prompt tiles and decodes whose keys several work-groups share, of few sequences and of more than a wave's lanes hold."""
    b = batch(rng, device, [(2500, 60), (0, 150), (1700, 33), (9, 0), (3100, 100)], H, KV)
    check(b, attend(b, device))
    check(b, attend(b, device, cut=False))
    b = batch(rng, device, [(int(c), 1) for c in rng.integers(0, 400, 150)] + [(9000, 1), (5000, 1)], 2 * H // H, 1)
    b["longest"] = 200000  # a hint: the sequences may be that long
    check(b, attend(b, device))


@pytest.mark.parametrize("cut", [True, False])
@pytest.mark.parametrize("H,KV", [(4, 2), (8, 1), (40, 2)])
def test_attention_of_steps_of_decodes_and_prompts(rng, device, H, KV, cut):
    """Many decodes, short runs and a few chunks in one call, told to be of long contexts."""
    new = [1] * 60 + [5, 90, 0, 17, 130, 16, 1]
    b = batch(rng, device, [(int(c), n) for c, n in zip(rng.integers(0, 500, len(new)), new)] + [(3000, 1), (2600, 70)], H, KV)
    b["longest"] = 30_000
    check(b, attend(b, device, cut=cut, pad=3))


def test_a_workspace_serves_calls_of_every_shape(rng, device):
    """Prompts, runs and decodes in turn with one workspace: each leaves it as the others, laid out otherwise, need it."""
    ws = K.kv4_workspace(200, 6, n_heads=8, n_kv=2, max_query=100, max_context=100_000, device=device)
    shapes = [[(6000, 100), (4500, 77)], [(9000, 1), (20, 1), (7000, 1)], [(5000, 5), (8000, 8)], [(3000, 1)] * 6]
    calls = []
    for seqs in shapes:
        b = batch(rng, device, seqs, 8, 2)
        out = torch.zeros(b["T"], 8, D, dtype=torch.float16, device=device)
        args = (on(b["q"], device), on(b["pages"], device), out, dint(b["start"], device), dint(b["pos"], device), dint(b["table"], device))
        calls.append((b, args))
    for b, args in calls * 2:
        args[2].fill_(7.0)
        K.kv4_attention(*args, max_query=b["most"], max_context=100_000, workspace=ws)
        check(b, args[2].double().cpu().numpy())


@pytest.mark.parametrize("S,H,KV", [(64, 16, 8), (47, 8, 8), (65, 10, 5), (200, 4, 2), (256, 2, 2), (170, 12, 2)])
def test_attention_dealt_by_length(rng, device, S, H, KV):
    """More items than CUs of contexts that may be long: many lengths alike, empty sequences, runs of several tokens."""
    seqs = [(int(c), int(n)) for c, n in zip(rng.choice([0, 16, 33, 150, 700], S), rng.choice([1, 1, 1, 0, 2], S))]
    seqs[S // 2] = 4000, 1
    b = batch(rng, device, seqs, H, KV)
    check(b, attend(b, device, pad=2))
    check(b, attend(b, device, cut=False))
    b["table"][3, 1:] = -1  # missing pages
    b["most"] = 1
    check(b, attend(b, device))
    # longer runs than the call was told of: entries of many tiles
    seqs = [(int(c), 1) for c in rng.integers(0, 300, S)]
    seqs[1] = seqs[S - 2] = 900, 300
    b = batch(rng, device, seqs, H, KV)
    b["most"], b["longest"] = 1, 260 * PAGE
    b["table"] = np.pad(b["table"], ((0, 0), (0, 260 - b["table"].shape[1])), constant_values=-1)
    b["W"] = 260
    check(b, attend(b, device))


def test_attention_of_more_sequences_than_a_launch_takes(rng, device):
    b = batch(rng, device, [(int(c), 1) for c in rng.integers(0, 40, 4200)], 1, 1)
    check(b, attend(b, device, pad=1))


def test_attention_without_hints_and_beyond_them(rng, device):
    b = batch(rng, device, [(100, 40), (700, 1)], 4, 2)
    check(b, attend(b, device, hints=False))
    for most, longest in ((1, 10), (3, 200), (40, 64), (8, 741)):
        b["most"], b["longest"] = most, longest
        check(b, attend(b, device))


def test_attention_of_empty_batches_and_negative_positions(rng, device):
    b = batch(rng, device, [(0, 0), (0, 0)], 4, 2)
    assert attend(b, device, pad=4).size == 0
    b = batch(rng, device, [(0, 3), (50, 2)], 4, 2)
    b["pos"][:3] = -1
    got = attend(b, device)
    assert (got[:3] == 0).all()
    check(b, got)


def test_attention_reads_missing_pages_as_zeros(rng, device):
    b = batch(rng, device, [(100, 1), (90, 5)], 4, 2)
    b["table"][0, 2] = -1
    b["table"][1, 3] = 10 ** 6
    got = attend(b, device)
    b["table"][1, 3] = -1
    check(b, got)


@pytest.mark.parametrize("new", [1, 9, 60])
def test_attention_scores_of_any_size(rng, device, new):
    """Scores far apart and far from zero; the largest keys that pages hold."""
    for spread, scale in ((1.0, 5.0), (100.0, 1.0), (8000.0, 0.5), (1e-4, 1e-6)):
        b = batch(rng, device, [(200, new), (17, new)], 4, 2, spread=spread)
        got = attend(b, device, scale=scale)
        assert np.isfinite(got).all()
        check(b, got, scale)


def test_attention_of_a_row_with_nan(rng, device):
    """A NaN in q makes that (token, head) NaN and no other."""
    for new in (1, 40):
        b = batch(rng, device, [(300, new), (20, new)], 4, 2)
        b["q"][0, 1, 5] = np.nan
        got = attend(b, device)
        assert np.isnan(got[0, 1]).all()
        other = np.ones(got.shape[:2], bool)
        other[0, 1] = False
        assert np.isfinite(got[other]).all()


def test_attention_of_a_pool_past_32_bits(rng, device):
    """Pages whose bytes lie beyond 2^32 (and 2^31 from one another)."""
    blocks, KV = 300_000, 8  # 5.2 GB
    pool = torch.zeros(blocks, KV, PAGE_BYTES, dtype=torch.uint8, device=device)
    b = batch(rng, device, [(150, 1), (100, 20)], 16, KV)
    at = np.sort(rng.permutation(blocks - 1)[: b["pages"].shape[0]])
    at[-3:] = blocks - 3, blocks - 2, blocks - 1
    at[:2] = 0, 125_000
    pool[on(at, device)] = on(b["pages"], device)
    table = np.where(b["table"] >= 0, at[b["table"]], -1)
    out = torch.zeros(b["T"], 16, D, dtype=torch.float16, device=device)
    K.kv4_attention(on(b["q"], device), pool, out, dint(b["start"], device), dint(b["pos"], device), dint(table, device))
    check(b, out.double().cpu().numpy())


def test_attention_keeps_a_nearly_equal_tail(rng, device):
    """Thousands of weights that f16 could not hold beside a largest weight of 1 still count."""
    n = 3000
    b = batch(rng, device, [(n, 1)], 1, 1)
    b["q"][:] = 0
    b["q"][0, 0, 0] = 1.0
    k = np.zeros((b["pages"].shape[0], 1, PAGE, D))
    v = np.ones_like(k)
    first = b["table"][0, 0]
    k[first, 0, 0, 0] = 6.0
    v[first, 0, 0] = 0.0
    b["pages"] = ref.to_pages(k, v)
    check(b, attend(b, device, scale=2.5), 2.5)  # weights e^-15 beside 1: 3000 of them are 9e-4


# ---- products ----

EPILOGUES = [_lib.EPILOGUE_STORE_F16, _lib.EPILOGUE_STORE_F32, _lib.EPILOGUE_ADD_F32, _lib.EPILOGUE_SILU_MUL]


def weights(rng, N, k, spread=6):
    """Codes and scales [N, k] at random, the scales over 2^spread."""
    codes = rng.integers(0, 256, (N, k // 2)).astype(np.uint8)
    return codes, rng.integers(124 - spread, 124, (N, k // 32)).astype(np.uint8)


def product(a, codes, scales, epilogue, c0=None):
    """The product in float64 and the bound on a kernel's: f32 sums of K exact terms (K + 16 roundings, the waves' sums
    and the epilogue's among them), silu's exponential, quotient and product (8 roundings and 2^-20), the f16 rounding."""
    w = ref.decode(ref.unpack(codes), scales)
    a = a.astype(np.float64)
    y, mass = a @ w.T, np.abs(a) @ np.abs(w).T
    e = (a.shape[1] + 16) * 2.0 ** -24 * mass
    if epilogue == _lib.EPILOGUE_STORE_F32:
        return y, e
    if epilogue == _lib.EPILOGUE_ADD_F32:
        return c0 + y, e + 2.0 ** -24 * (np.abs(c0) + np.abs(y))
    if epilogue == _lib.EPILOGUE_SILU_MUL:
        g, u, eg, eu = y[:, ::2], y[:, 1::2], e[:, ::2], e[:, 1::2]
        with np.errstate(over="ignore"):
            s = 1 / (1 + np.exp(-g))
        y = g * s * u
        # |d silu / dg| <= 1.1
        e = 1.1 * eg * (np.abs(u) + eu) + np.abs(g * s) * eu + (8 * 2.0 ** -24 + 2.0 ** -20) * np.abs(y)
    lim = 65504.0
    return np.clip(y, -lim, lim), e + 2.0 ** -11 * (np.abs(y) + e) + 2.0 ** -25


def run_product(rng, device, a, codes, scales, epilogue, wide=0):
    N = codes.shape[0]
    cols = N // 2 if epilogue == _lib.EPILOGUE_SILU_MUL else N
    f32 = epilogue in (_lib.EPILOGUE_STORE_F32, _lib.EPILOGUE_ADD_F32)
    c0 = rng.standard_normal((a.shape[0], cols)).astype(np.float32) if f32 else None
    c = torch.full((a.shape[0], cols + wide), 5.0, dtype=torch.float32 if f32 else torch.float16, device=device)
    if f32:
        c[:, :cols] = on(c0, device)
    w = K.gemv4_pack(on(codes, device), on(scales, device))
    ad = torch.full((a.shape[0], a.shape[1] + 8 * wide), float("nan"), dtype=torch.float16, device=device)
    ad[:, : a.shape[1]] = on(a, device)
    K.gemv4(ad[:, : a.shape[1]], w, c[:, :cols], epilogue, N=N)
    assert (c[:, cols:] == 5).all()
    want, bound = product(a, codes, scales, epilogue, c0)
    got = c[:, :cols].double().cpu().numpy()
    assert (np.abs(got - want) <= bound).all()
    return c[:, :cols].clone()


@pytest.mark.parametrize("epilogue", EPILOGUES)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 33, 64, 65, 130, 200])
def test_products_of_all_rows(rng, device, M, epilogue):
    codes, scales = weights(rng, 50, 1056)
    a = rng.standard_normal((M, 1056)).astype(np.float16)
    run_product(rng, device, a, codes, scales, epilogue, wide=3)


@pytest.mark.parametrize("epilogue", EPILOGUES)
@pytest.mark.parametrize("N,k", [(2, 32), (16, 64), (18, 96), (34, 128), (128, 160), (1000, 1024), (4096, 2080), (66, 12288)])
@pytest.mark.parametrize("M", [1, 20, 100])
def test_products_of_all_shapes(rng, device, M, N, k, epilogue):
    codes, scales = weights(rng, N, k)
    run_product(rng, device, rng.standard_normal((M, k)).astype(np.float16), codes, scales, epilogue)


@pytest.mark.parametrize("N", [1, 17, 151, 70001])
def test_products_of_odd_feature_counts(rng, device, N):
    codes, scales = weights(rng, N, 256)
    run_product(rng, device, rng.standard_normal((3, 256)).astype(np.float16), codes, scales, _lib.EPILOGUE_STORE_F32, wide=1)


@pytest.mark.parametrize("N,k", [(48, 1056), (4096, 2048), (70000, 512), (300, 4096), (200, 6144), (2100, 6144), (100, 8992)])
def test_a_row_has_the_same_bits_in_every_batch(rng, device, N, k):
    codes, scales = weights(rng, N, k)
    w = K.gemv4_pack(on(codes, device), on(scales, device))
    a = on(rng.standard_normal((300, k)).astype(np.float16), device)
    one = torch.empty(1, N, device=device)
    K.gemv4(a[7:8], w, one, _lib.EPILOGUE_STORE_F32, N=N)
    for rows in (8, 16, 17, 33, 64, 65, 128, 129, 300):
        c = torch.empty(rows, N, device=device)
        K.gemv4(a[:rows], w, c, _lib.EPILOGUE_STORE_F32, N=N)
        assert torch.equal(c[7], one[0]), rows


def test_products_of_more_rows_than_a_launch_takes(rng, device):
    codes, scales = weights(rng, 2, 32)
    w = K.gemv4_pack(on(codes, device), on(scales, device))
    a = torch.randn(1 << 21, 32, device=device).half()
    c = torch.zeros(1 << 21, 2, device=device)
    K.gemv4(a, w, c, _lib.EPILOGUE_STORE_F32, N=2)
    for rows in (slice(0, 40), slice((1 << 20) - 20, (1 << 20) + 20), slice((1 << 21) - 40, None)):
        want, bound = product(a[rows].double().cpu().numpy(), codes, scales, _lib.EPILOGUE_STORE_F32)
        assert (np.abs(c[rows].double().cpu().numpy() - want) <= bound).all()


def test_products_keep_special_values_in_their_places(rng, device):
    """NaN and infinity in a row of A or in a weight's group reach that row or feature and no other; large outputs clamp."""
    codes, scales = weights(rng, 40, 96)
    codes[:] = codes & 0x77  # no signs, so that an infinity stays one
    codes |= 0x22
    a = np.ones((5, 96), np.float16)
    a[1, 95], a[3, 2] = np.nan, np.inf
    scales[7, 1] = 255
    w = K.gemv4_pack(on(codes, device), on(scales, device))
    c = torch.empty(5, 40, device=device)
    K.gemv4(on(a, device), w, c, _lib.EPILOGUE_STORE_F32, N=40)
    c = c.cpu().numpy()
    feature = np.arange(40) != 7
    assert np.isnan(c[1]).all() and np.isnan(c[:, 7]).all()
    assert (c[3, feature] == np.inf).all() and np.isfinite(c[np.ix_([0, 2, 4], np.nonzero(feature)[0])]).all()
    scales[:] = 140
    h = torch.empty(2, 40, dtype=torch.float16, device=device)
    K.gemv4(on(np.float16([[1] * 96, [-1] * 96]), device), K.gemv4_pack(on(codes, device), on(scales, device)), h, _lib.EPILOGUE_STORE_F16, N=40)
    assert (h[0] == 65504).all() and (h[1] == -65504).all()


def test_pack_is_the_documented_layout(rng, device):
    codes, scales = weights(rng, 21, 160)
    got = K.gemv4_pack(on(codes, device), on(scales, device)).cpu().numpy()
    want = np.zeros((2, 2, 1088), np.uint8)
    for n in range(21):
        for j in range(5):
            for g in range(4):
                at = 16 * (16 * g + n % 16) + 4 * (j % 4)
                want[n // 16, j // 4, at:at + 4] = codes[n, 16 * j + 4 * g:16 * j + 4 * g + 4]
            want[n // 16, j // 4, 1024 + 4 * (n % 16) + j % 4] = scales[n, j]
    assert np.array_equal(got, want.reshape(-1))


# ---- together ----

def test_python_refusals(device):
    pool = K.kv4_pool(4, 2, device)
    z = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    i = lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    ok = dict(q=z(3, 4, D), pool=pool, out=z(3, 4, D), query_start=i(3), positions=i(3), block_tables=i(2, 4))
    K.kv4_attention(**ok)
    for name, bad, text in [("q", z(3, 4, D, dtype=torch.float32), "f16"), ("pool", pool.view(torch.int8), "pool"), ("pool", pool[:, :, :100].contiguous(), "pool"),
                            ("pool", pool.view(-1), "pool"), ("out", z(3, 4, D, dtype=torch.float32), "out"), ("out", z(2, 4, D), "out"),
                            ("q", z(3, D, 4).transpose(1, 2), "q must"), ("positions", i(2), "positions"), ("block_tables", i(1, 4), "block_tables"),
                            ("query_start", z(3, dtype=torch.int64), "query_start")]:
        with pytest.raises(EmberError, match=text):
            K.kv4_attention(**{**ok, name: bad})
    with pytest.raises(EmberError, match="max_context"):
        K.kv4_attention(**ok, max_context=0)
    with pytest.raises(EmberError, match="do not group"):
        K.kv4_attention(**{**ok, "q": z(3, 3, D), "out": z(3, 3, D)})
    f = z(64, dtype=torch.float32)
    a = dict(qkv=z(3, 8 * D), q_out=z(3, 4 * D), pool=pool, positions=i(3), token_seq=i(3), block_tables=i(1, 4), n_heads=4, n_kv=2, inv_freq_dev=f)
    K.kv4_append(**a)
    for name, bad, text in [("qkv", z(2, 8 * D), "as many tokens"), ("q_out", z(3, 3 * D), "as many"), ("token_seq", i(2), "as many"),
                            ("block_tables", i(4), "block_tables"), ("inv_freq_dev", f[:32], "64 values"), ("n_kv", 1, "as many"),
                            ("q_norm", z(D, dtype=torch.float32), "go together"), ("k_out", z(3, 2 * D), "go together"), ("k_out", z(3, D), "k_out"),
                            ("bias", z(7, dtype=torch.float32), "bias"), ("qkv", z(3, 16 * D)[:, ::2], "qkv"), ("pool", K.kv4_pool(4, 3, device), "n_kv heads")]:
        with pytest.raises(EmberError, match=text):
            K.kv4_append(**{**a, name: bad})
    for bad in (z(4, 48), z(4), z(4, 64).t(), z(4, 64, dtype=torch.bfloat16)):
        with pytest.raises(EmberError, match="mx_quantize"):
            K.mx_quantize(bad)
    codes, scales = K.mx_quantize(z(16, 64))
    for c, s in ((codes, scales[:, :1]), (codes.t(), scales), (codes, scales.int())):
        with pytest.raises(EmberError):
            K.gemv4_pack(c, s)
    w = K.gemv4_pack(codes, scales)
    K.gemv4(z(2, 64), w, z(2, 16), _lib.EPILOGUE_STORE_F16, N=16)
    for x, c, n in ((z(2, 160), z(2, 16), 16), (z(2, 64), z(2, 15), 16), (z(2, 64), z(2, 16), 17), (z(2, 64, dtype=torch.float32), z(2, 16), 16),
                    (z(64, 2).t(), z(2, 16), 16), (z(2, 64), z(2, 16, dtype=torch.float32), 16), (z(2, 68)[:, :64], z(2, 16), 16)):
        with pytest.raises(EmberError):
            K.gemv4(x, w, c, _lib.EPILOGUE_STORE_F16, N=n)
    with pytest.raises(EmberError, match="epilogue"):
        K.gemv4(z(2, 64), w, z(2, 16), 9, N=16)


def four_bit_step(device, t, state, stream=None):
    """RMSNorm, 4-bit qkv projection, append, attention, 4-bit output projection into the residual."""
    H, KV, hid = state["H"], state["KV"], state["hid"]
    K.rmsnorm_rows(state["x"], state["norm"], state["xn"], 1e-6, stream=stream)
    K.gemv4(state["xn"], state["wqkv"], state["qkv"], _lib.EPILOGUE_STORE_F16, N=(H + 2 * KV) * D, stream=stream)
    K.kv4_append(state["qkv"], state["q"], state["pool"], t.positions, t.token_seq, t.block_tables, n_heads=H, n_kv=KV,
                 inv_freq_dev=state["freq"], q_norm=state["qn"], k_norm=state["kn"], stream=stream)
    K.kv4_attention(state["q"].view(-1, H, D), state["pool"], state["attn"].view(-1, H, D), t.query_start, t.positions, t.block_tables,
                    max_query=state["most"], max_context=300, workspace=state["ws"], stream=stream)
    K.gemv4(state["attn"], state["wo"], state["x"], _lib.EPILOGUE_ADD_F32, N=hid, stream=stream)


def make_step(rng, device, new, cached, rows):
    H, KV, hid, S, W = 8, 4, 256, len(new), 24
    g = lambda *s: on(rng.standard_normal(s).astype(np.float32), device)  # noqa: E731
    pack = lambda w: K.gemv4_pack(*K.mx_quantize(w))  # noqa: E731
    blocks = S * W
    st = dict(H=H, KV=KV, hid=hid, most=max(new), norm=g(hid), freq=on(K.inv_freq(1e4), device), qn=g(D), kn=g(D),
              wqkv_f=g((H + 2 * KV) * D, hid) / 16, wo_f=g(hid, H * D) / 32, x0=g(rows, hid))
    k, v = rng.standard_normal((2, blocks + 1, KV, PAGE, D))
    st["pages0"] = ref.to_pages(k, v)
    f16 = lambda n: torch.zeros(rows, n, dtype=torch.float16, device=device)  # noqa: E731
    st.update(wqkv=pack(st["wqkv_f"]), wo=pack(st["wo_f"]), x=st["x0"].clone(), xn=f16(hid), qkv=f16((H + 2 * KV) * D), q=f16(H * D),
              attn=f16(H * D), pool=on(st["pages0"], device),
              ws=K.kv4_workspace(rows, S, n_heads=H, n_kv=KV, max_query=max(new), max_context=300, device=device))
    t = K.StepTables(S, rows, W, device)
    request = np.full((S, W), -1)
    for s, c in enumerate(cached):
        n = -(-c // PAGE)
        request[s, :n] = s * W + np.arange(n)
    K.step_tables(t, dint(request, device), dint(cached, device), dint(new, device),
                  dint([s * W + i for s in range(S) for i in range(-(-cached[s] // PAGE), -(-(cached[s] + new[s]) // PAGE))], device),
                  pad_block=blocks)
    return t, st


def step_reference(t, st, rows):
    """The same step in float64 over the same 4-bit weights and pages; q and the codes from the kernels' own f16 qkv."""
    w = lambda x: ref.decode(*[f(y.cpu().numpy()) for f, y in zip((ref.unpack, lambda z: z), K.mx_quantize(x))])  # noqa: E731
    H, KV = st["H"], st["KV"]
    x = st["x0"].double().cpu().numpy()
    xn = st["norm"].double().cpu().numpy() * x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
    T = int(t.totals[0])
    pos, seq, table = (getattr(t, n).cpu().numpy() for n in ("positions", "token_seq", "block_tables"))
    qkv = st["qkv"].double().cpu().numpy()
    k, v = ref.read_pages(st["pool"].cpu().numpy())
    q = st["q"].cpu().numpy().reshape(rows, H, D)[:T]
    attn, bound = attention_reference(q, k, v, table[:-1], t.query_start.cpu().numpy(), pos, lambda s, p, j: j <= p, True)
    return xn @ w(st["wqkv_f"]).T, qkv, attn, bound, w(st["wo_f"]), x


@pytest.mark.parametrize("new,cached", [([1, 1, 1, 1], [0, 15, 200, 99]), ([3, 1, 0, 5], [20, 299, 7, 31]), ([60, 1, 40], [0, 64, 130])])
def test_a_step_in_four_bits(rng, device, new, cached):
    rows = sum(new) + 3
    t, st = make_step(rng, device, new, cached, rows)
    four_bit_step(device, t, st)
    T = int(t.totals[0])
    assert T == sum(new) and int(t.totals[2]) == 0
    qkv, got_qkv, attn, bound, wo, x = step_reference(t, st, rows)
    # f16 activations (the norm's, 2^-11) through 256 products of 4-bit weights, and qkv's own rounding
    slack = 2.0 ** -11 * (np.abs(qkv) + np.sqrt(256) * np.abs(qkv).std()) * 4
    assert (np.abs(got_qkv - qkv) <= slack).all()
    got = st["attn"].double().cpu().numpy().reshape(rows, st["H"], D)[:T]
    assert (np.abs(got - attn) <= bound).all()
    flat = st["attn"].double().cpu().numpy()
    out = st["x"].double().cpu().numpy()
    e = (wo.shape[1] + 16) * 2.0 ** -24 * (np.abs(flat) @ np.abs(wo).T) + 2.0 ** -22 * (np.abs(x) + np.abs(flat @ wo.T))
    assert (np.abs(out - (x + flat @ wo.T)) <= e)[:T].all()
    # untouched slots keep their bytes
    pages = st["pool"].cpu().numpy()
    tokens = {(int(b), int(s)) for b, s in zip(t.slots[:T].cpu().numpy() // PAGE, t.slots[:T].cpu().numpy() % PAGE)}
    tokens.add((pages.shape[0] - 1, 0))  # the padding rows' slot
    k0, v0 = ref.read_pages(st["pages0"])
    k1, v1 = ref.read_pages(pages)
    for b in range(pages.shape[0]):
        for s in range(PAGE):
            if (b, s) not in tokens:
                assert np.array_equal(k0[b, :, s], k1[b, :, s]) and np.array_equal(v0[b, :, s], v1[b, :, s])


def test_a_step_in_four_bits_captured_and_replayed(rng, device):
    t, st = make_step(rng, device, [1, 1, 1, 1, 1], [0, 15, 200, 99, 290], 8)
    four_bit_step(device, t, st)
    eager = {n: st[n].clone() for n in ("x", "attn", "pool")}
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        four_bit_step(device, t, st)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            four_bit_step(device, t, st)
    for _ in range(4):
        st["x"].copy_(st["x0"])
        st["attn"].fill_(3)
        st["pool"].copy_(on(st["pages0"], device))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(st["pool"][:-1], eager["pool"][:-1])  # the last page: three padding rows write one slot
        for n in ("x", "attn"):  # the padding's rows of attn are left as they were, and x's so depend on them
            assert torch.equal(st[n][:5], eager[n][:5]), n


def test_long_contexts_captured_and_replayed(rng, device):
    """A prompt's tiles and long decodes, shared out by many work-groups, in one graph with one workspace; eager calls with
    another between its replays."""
    shapes = [batch(rng, device, seqs, 8, 2) for seqs in ([(6000, 100), (2000, 77)], [(9000, 1), (7000, 1), (0, 0)])]
    calls = [((on(b["q"], device), on(b["pages"], device), torch.zeros(b["T"], 8, D, dtype=torch.float16, device=device),
               *(dint(b[n], device) for n in ("start", "pos", "table"))), dict(max_query=b["most"], max_context=b["longest"])) for b in shapes]
    own, other = (K.kv4_workspace(200, 3, n_heads=8, n_kv=2, max_query=100, max_context=10_000, device=device) for _ in range(2))
    eager = []
    for b, (args, hints) in zip(shapes, calls):
        K.kv4_attention(*args, **hints, workspace=other)
        check(b, args[2].double().cpu().numpy())
        eager.append(args[2].clone())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for args, hints in calls:
            K.kv4_attention(*args, **hints, workspace=own)
    for _ in range(4):
        for args, _ in calls:
            args[2].fill_(7.0)
        graph.replay()
        for (args, hints), want in zip(calls, eager):
            assert torch.equal(args[2], want)
            K.kv4_attention(*args, **hints, workspace=other)
            assert torch.equal(args[2], want)


def test_calls_on_another_stream(rng, device):
    """Two streams at once, a workspace each."""
    a, b = batch(rng, device, [(900, 1), (30, 1)], 4, 2), batch(rng, device, [(500, 3)], 4, 2)
    calls = []
    for x in (a, b):
        s = torch.cuda.Stream()
        out = torch.zeros(x["T"], 4, D, dtype=torch.float16, device=device)
        ws = K.kv4_workspace(x["T"], len(x["start"]) - 1, n_heads=4, n_kv=2, max_query=x["most"], max_context=x["longest"], device=device)
        calls.append((x, s, out, ws, (on(x["q"], device), on(x["pages"], device), out, dint(x["start"], device), dint(x["pos"], device), dint(x["table"], device))))
    torch.cuda.synchronize()
    for _ in range(20):
        for x, s, out, ws, args in calls:
            K.kv4_attention(*args, max_query=x["most"], max_context=x["longest"], workspace=ws, stream=s)
    torch.cuda.synchronize()
    for x, s, out, ws, args in calls:
        check(x, out.double().cpu().numpy())


def test_preparation_on_another_stream(rng, device):
    """What mx_quantize and gemv4_pack return on a stream, given as an object or a handle, is theirs from the start."""
    x = on(rng.standard_normal((300, 256)).astype(np.float32), device)
    codes, scales = K.mx_quantize(x)
    packed = K.gemv4_pack(codes, scales)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        c, e = K.mx_quantize(x, stream=stream)
        w = K.gemv4_pack(c, e, stream=stream)
        s.synchronize()
        assert torch.equal(c, codes) and torch.equal(e, scales) and torch.equal(w, packed)
