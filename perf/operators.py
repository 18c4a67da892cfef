"""Step tables on the GPU, windowed attention and shared-prefix attention, as cases that are measured.

Three operators of a serving step over the paged KV cache. Sizes are the benchmark's and the tests': decode at batch 32
over 256 to 4096 tokens, speculative verify at batch 64, 512-token prompt chunks, 2000 tokens on a 14,000-token
document, 256 sequences, 1024-token shared prefixes, 16 query and 8 kv heads of 128 (and the other head layouts of the
tests), pages of 16 tokens.

  tables   request lengths to a step's integers: query_start, positions, token_seq, slots, block tables, pages taken.
  window   attention of each token to the last `window` tokens and the first `sinks` ones; pages in between are freed.
  prefix   attention of groups of sequences that share a cached prefix, read once for the group.

Sequence lengths come from the case alone (its `lens`), values and page places from the seed. With ``own`` true ``run``
calls ``ember_amd.kernels``, else it computes the same in elementary torch operations.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE, D = 16, 128

TABLES = dict(op="tables", requests=64, seqs=32, max_blocks=256, ctx_lo=256, ctx_hi=4000, chunks=0, chunk=0, verify=1,
              lens=1)
WINDOW = dict(op="window", seqs=1, new=1, ragged=False, ctx_lo=640, ctx_hi=640, window=512, sinks=4, heads=16,
              kv_heads=8, dtype="f16", strided=False, lens=1)
PREFIX = dict(op="prefix", groups=1, seqs=8, new=1, prefix_lo=1024, prefix_hi=1024, own_lo=16, own_hi=256, whole=True,
              heads=16, kv_heads=8, dtype="f16", lens=1)


def listed() -> list:
    return [
        # A decode batch's tables: 32 of 64 known requests, one new token each. All latency.
        dict(name="tables_decode_b32", **TABLES),
        # A full card's step: 1000 of 1500 requests with up to 32,768 tokens each, 40 of them a 512-token prompt chunk.
        dict(name="tables_mixed_b1000", **{**TABLES, **dict(requests=1500, seqs=1000, max_blocks=2048, ctx_lo=64,
                                                            ctx_hi=32000, chunks=40, chunk=512, verify=5, lens=2)}),
        # One user's chat turn with a short window: the smallest call.
        dict(name="window_decode_b1", **WINDOW),
        # Batched decode of long conversations, each reading 4096 recent tokens and the first 4.
        dict(name="window_decode_b32", **{**WINDOW, **dict(seqs=32, ctx_lo=300, ctx_hi=16384, window=4096, lens=3)}),
        # Speculative verify with 1 to 5 tokens a sequence, q a part of the projection's rows.
        dict(name="window_verify_b64", **{**WINDOW, **dict(seqs=64, new=5, ragged=True, ctx_lo=512, ctx_hi=4096,
                                                           window=1000, sinks=64, strided=True, lens=4)}),
        # Prompt chunks of up to 512 tokens of 4 requests.
        dict(name="window_prompt_4x512", **{**WINDOW, **dict(seqs=4, new=512, ragged=True, ctx_lo=900, ctx_hi=3000,
                                                             window=1024, sinks=16, lens=5)}),
        # A long document's chunk: 2000 tokens on a 12,000-token context with a wide window.
        dict(name="window_prompt_2000", **{**WINDOW, **dict(seqs=1, new=2000, ctx_lo=12000, ctx_hi=12000, window=4096,
                                                            sinks=4, lens=6)}),
        # The f32 parity path: a few sequences, one short of its window.
        dict(name="window_f32_b5", **{**WINDOW, **dict(seqs=5, new=3, ragged=True, ctx_lo=100, ctx_hi=1500, window=333,
                                                       sinks=5, heads=12, kv_heads=4, dtype="f32", lens=7)}),
        # Eight parallel samples of one prompt.
        dict(name="prefix_b8_1024", **PREFIX),
        # A system prompt of 8000 tokens in front of 64 conversations.
        dict(name="prefix_b64_8000", **{**PREFIX, **dict(seqs=64, prefix_lo=8000, prefix_hi=8000, own_lo=30,
                                                         own_hi=1500, heads=32, lens=8)}),
        # 256 decodes behind 16 prompts of their own, the last page of a prompt copied for each.
        dict(name="prefix_b256_16groups", **{**PREFIX, **dict(groups=16, seqs=256, prefix_lo=500, prefix_hi=4096,
                                                              own_lo=1, own_hi=700, whole=False, lens=9)}),
        # Verify of 3 tokens a sequence on the f32 path.
        dict(name="prefix_f32_b6", **{**PREFIX, **dict(groups=2, seqs=6, new=3, prefix_lo=130, prefix_hi=900, own_lo=1,
                                                       own_hi=90, whole=False, heads=4, kv_heads=2, dtype="f32",
                                                       lens=10)}),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(16, 8), (16, 8), (32, 8), (8, 8), (12, 4), (4, 2), (8, 1)]


def _draw_one(rng: random.Random) -> dict:
    op = rng.choice(["tables", "window", "window", "window", "prefix", "prefix"])
    lens = rng.randrange(1 << 20)
    if op == "tables":
        seqs = _log_int(rng, 1, 1000)
        blocks = _log_int(rng, 40, 2048)
        hi = _log_int(rng, 20, blocks * PAGE - 520)
        return {**TABLES, **dict(requests=seqs + _log_int(rng, 1, 500), seqs=seqs, max_blocks=blocks,
                                 ctx_lo=rng.randint(0, hi), ctx_hi=hi, chunks=rng.randint(0, min(seqs, 40)),
                                 chunk=_log_int(rng, 2, 512), verify=rng.randint(1, 6), lens=lens)}
    heads, kv = rng.choice(HEADS)
    dtype = "f32" if rng.random() < 0.2 else "f16"
    if op == "window":
        kind = rng.choice(["decode", "verify", "prompt"])
        if kind == "prompt":
            seqs, new = _log_int(rng, 1, 6), _log_int(rng, 6, 2000 if dtype == "f16" else 100)
        else:
            seqs, new = _log_int(rng, 1, 128), 1 if kind == "decode" else rng.randint(2, 8)
        hi = _log_int(rng, 1, 16384)
        return {**WINDOW, **dict(seqs=seqs, new=new, ragged=rng.random() < 0.5, ctx_lo=rng.randint(0, hi), ctx_hi=hi,
                                 window=_log_int(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 16, 50, 130]), heads=heads,
                                 kv_heads=kv, dtype=dtype, strided=rng.random() < 0.3, lens=lens)}
    groups = _log_int(rng, 1, 16)
    seqs = max(groups, _log_int(rng, 1, 256))
    hi = _log_int(rng, 1, 8192 if seqs <= 64 else 4096)
    own_hi = _log_int(rng, 1, 1500)
    return {**PREFIX, **dict(groups=groups, seqs=seqs, new=rng.choice([1, 1, 1, 2, 5]), prefix_lo=rng.randint(1, hi),
                             prefix_hi=hi, own_lo=rng.randint(1, own_hi), own_hi=own_hi, whole=rng.random() < 0.5,
                             heads=heads, kv_heads=kv, dtype=dtype, lens=lens)}


def draw(rng: random.Random) -> dict:
    top = {}
    for c in listed():
        w = work(c)
        for k in w:
            top[c["op"], k] = max(top.get((c["op"], k), 0), w[k])
    while True:
        c = _draw_one(rng)
        w = work(c)
        # an f32 case computes outside the matrix units: it stays with a tenth of the largest work
        cut = 10 if c.get("dtype") == "f32" else 1
        if all(w[k] * cut <= top[c["op"], k] for k in w) and _memory(c) < 12e9:
            return c


# ---- lengths, from the case alone ----

def _lens(case: dict) -> dict:
    """Host arrays: per sequence the cached tokens and the new ones; for prefix also groups and prefix lengths."""
    r = np.random.RandomState(case["lens"])
    S = case["seqs"]
    if case["op"] == "tables":
        cached = r.randint(case["ctx_lo"], case["ctx_hi"] + 1, S)
        new = r.randint(1, case["verify"] + 1, S)
        at = r.permutation(S)[: case["chunks"]]
        new[at] = r.randint(1, max(2, case["chunk"]) + 1, at.size) if case["chunks"] else 0
        if S > 4:
            new[r.randint(0, S, S // 5)] = 0  # requests that wait in this step
        return dict(cached=cached, new=new, request=r.permutation(case["requests"])[:S])
    new = np.full(S, case["new"])
    if case["op"] == "window":
        cached = r.randint(case["ctx_lo"], case["ctx_hi"] + 1, S)
        if case["ragged"]:
            new = r.randint(1, case["new"] + 1, S)
        return dict(cached=cached, new=new)
    G = case["groups"]
    # every group holds one sequence or more
    start = np.concatenate([[0], np.sort(r.permutation(S - 1)[: G - 1]) + 1, [S]]) if G > 1 else np.array([0, S])
    prefix = r.randint(case["prefix_lo"], case["prefix_hi"] + 1, G)
    if case["whole"]:
        prefix = np.maximum(PAGE, prefix // PAGE * PAGE)
    own_keys = r.randint(case["own_lo"], case["own_hi"] + 1, S)  # behind the prefix, the new tokens among them
    own_keys = np.maximum(own_keys, new)
    group = np.repeat(np.arange(G), np.diff(start))
    return dict(cached=prefix[group] + own_keys - new, new=new, start=start, prefix=prefix, group=group)


def _window_keys(case: dict, n: dict):
    """Per sequence: keys that some token sees, and (token, key) pairs that are visible."""
    w, k = case["window"], case["sinks"]
    keys, pairs = [], []
    for c, m in zip(n["cached"].tolist(), n["new"].tolist()):
        lo = max(0, c - w + 1)
        keys.append(c + m - lo + min(k, lo))
        p = np.arange(c, c + m)
        near = np.minimum(p + 1, w)
        pairs.append(int((near + np.minimum(k, p + 1 - near)).sum()))
    return np.array(keys), np.array(pairs)


def work(case: dict) -> dict:
    n = _lens(case)
    T = int(n["new"].sum())
    if case["op"] == "tables":
        S, W = case["seqs"], case["max_blocks"]
        used = int(((n["cached"] + PAGE - 1) // PAGE).sum())
        taken = int(((n["cached"] + n["new"] + PAGE - 1) // PAGE).sum()) - used
        cap = _capacity(case, n)
        return {"bytes": 4 * (3 * S + used + taken) + 4 * ((S + 1) * W + taken + 2 * (S + 1) + 4) + 16 * cap,
                "flops": 0}
    size = 2 if case["dtype"] == "f16" else 4
    token = 2 * T * case["heads"] * D * size
    if case["op"] == "window":
        keys, pairs = _window_keys(case, n)
        return {"bytes": int(keys.sum()) * case["kv_heads"] * D * 2 * size + token,
                "flops": 4 * D * case["heads"] * int(pairs.sum())}
    ctx = n["cached"] + n["new"]
    keys = int(n["prefix"].sum()) + int((ctx - n["prefix"][n["group"]]).sum())
    pairs = int((n["new"] * n["cached"] + n["new"] * (n["new"] + 1) // 2).sum())
    return {"bytes": keys * case["kv_heads"] * D * 2 * size + token, "flops": 4 * D * case["heads"] * pairs}


def _memory(case: dict) -> float:
    """Bytes of the plain form's largest tensors."""
    if case["op"] == "tables":
        return 8.0 * case["seqs"] * case["max_blocks"]
    n = _lens(case)
    S, M = case["seqs"], int(n["new"].max())
    L = (M + case["window"] + case["sinks"]) if case["op"] == "window" else int((n["cached"] + n["new"]).max())
    return 4.0 * S * L * (2 * case["kv_heads"] * D + 2 * case["heads"] * M)


def _capacity(case: dict, n: dict) -> int:
    """The token buffers' rows: the step's tokens up to the next 64, as a program that pads its steps has them."""
    return -(-max(1, int(n["new"].sum())) // 64) * 64


# ---- inputs ----

def prepare(case: dict, seed: int) -> dict:
    n = _lens(case)
    r = np.random.RandomState(seed % (1 << 31))
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    ints = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    S = case["seqs"]
    ctx = n["cached"] + n["new"]
    if case["op"] == "tables":
        R, W = case["requests"], case["max_blocks"]
        have = (n["cached"] + PAGE - 1) // PAGE
        need = int(((ctx + PAGE - 1) // PAGE - have).sum())
        blocks = int(have.sum()) + need + 8
        place = r.permutation(blocks)
        table = np.full((R, W), -1, np.int32)
        rows = np.repeat(n["request"], have)
        first = np.cumsum(have) - have
        cols = np.arange(int(have.sum())) - np.repeat(first, have)
        table[rows, cols] = place[: int(have.sum())]
        cached = r.randint(0, 100, R)  # requests that are not in this step have lengths too
        cached[n["request"]] = n["cached"]
        cursor = int(r.randint(0, 5))
        s = dict(case=case, request=ints(n["request"]), cached=ints(cached), new=ints(n["new"]), table=ints(table),
                 free=ints(np.concatenate([r.randint(0, blocks, cursor), place[int(have.sum()):]])),
                 cursor=ints([cursor]), capacity=_capacity(case, n), pad_block=blocks, blocks=blocks + 1)
        if own:
            from ember_amd import kernels as K
            s["out"] = K.StepTables(S, s["capacity"], W, device=dev)
        return s
    W = int((ctx.max() + PAGE - 1) // PAGE) + 1
    pages = (ctx + PAGE - 1) // PAGE
    table = np.full((S, W), -1, np.int32)
    copies = None
    if case["op"] == "window":
        lo = np.maximum(0, n["cached"] - case["window"] + 1) // PAGE  # the first page still needed
        head = -(-case["sinks"] // PAGE)
        col = np.arange(W)[None, :]
        live = (col < pages[:, None]) & ((col >= lo[:, None]) | (col < head))
        total = int(live.sum())
        blocks = total + 7
        table[live] = r.permutation(blocks)[:total]
    else:
        shared = n["prefix"] // PAGE  # whole pages of each group's prefix
        gs, ss = int(shared.sum()), pages - shared[n["group"]]
        blocks = gs + int(ss.sum()) + 7
        place = r.permutation(blocks)
        first = np.cumsum(shared) - shared
        col = np.arange(W)[None, :]
        sh = shared[n["group"]][:, None]
        table = np.where(col < sh, place[np.minimum(first[n["group"]][:, None] + col, blocks - 1)], table)
        mine = gs + (np.cumsum(ss) - ss)[:, None] + col - sh
        table = np.where((col >= sh) & (col < pages[:, None]), place[np.clip(mine, 0, blocks - 1)], table)
        rest = (n["prefix"] % PAGE)[n["group"]]
        head_seq = n["start"][:-1][n["group"]]
        sel = rest > 0
        copies = (table[head_seq, shared[n["group"]]][sel], table[np.arange(S), shared[n["group"]]][sel], rest[sel])
    T, H, KV = int(n["new"].sum()), case["heads"], case["kv_heads"]
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32
    k = torch.empty(blocks, KV, PAGE, D, dtype=dt, device=dev).normal_(generator=g)
    v = torch.empty(blocks, KV, PAGE, D, dtype=dt, device=dev).normal_(generator=g)
    if copies is not None and copies[0].size:  # the prompt's last, partial page stands in every sequence's own page
        src, dst, rest = (torch.from_numpy(np.ascontiguousarray(a, np.int64)).to(dev) for a in copies)
        keep = (torch.arange(PAGE, device=dev)[None, :] < rest[:, None])[:, None, :, None]
        k[dst] = torch.where(keep, k[src], k[dst])
        v[dst] = torch.where(keep, v[src], v[dst])
    row = (H + 2 * KV) * D if case.get("strided") else H * D
    q = (1.5 * torch.empty(T, row, device=dev).normal_(generator=g)).to(dt)[:, : H * D].view(T, H, D)
    start = np.concatenate([[0], np.cumsum(n["new"])])
    pos = np.repeat(n["cached"] - start[:-1], n["new"]) + np.arange(T)
    s = dict(case=case, q=q, k=k, v=v, table=ints(table), start=ints(start), pos=ints(pos), most=int(n["new"].max()),
             longest=int(ctx.max()))
    if case["op"] == "prefix":
        s.update(group_start=ints(n["start"]), prefix=ints(n["prefix"]), group=ints(n["group"]),
                 hints=dict(max_query=s["most"], max_prefix=int(n["prefix"].max()),
                            max_own=int((ctx - n["prefix"][n["group"]]).max()),
                            max_group=int(np.add.reduceat(n["new"], n["start"][:-1]).max())))
    if own:
        from ember_amd import kernels as K
        s["out"] = torch.empty(T, H, D, dtype=dt, device=dev)
        if case["op"] == "window":
            s["workspace"] = K.window_workspace(T, S, n_heads=H, n_kv=KV, window=case["window"], sinks=case["sinks"],
                                                max_query=s["most"], dtype=dt, device=dev)
        else:
            s["workspace"] = K.shared_prefix_workspace(T, S, case["groups"], n_heads=H, n_kv=KV, dtype=dt, device=dev,
                                                       **s["hints"])
    return s


# ---- the operators ----

def run(s: dict):
    c = s["case"]
    if own:
        from ember_amd import kernels as K
        if c["op"] == "tables":
            t = K.step_tables(s["out"], s["table"], s["cached"], s["new"], s["free"], request=s["request"],
                              free_cursor=s["cursor"], pad_block=s["pad_block"])
            return dict(query_start=t.query_start, context_len=t.context_len, positions=t.positions,
                        token_seq=t.token_seq, slots=t.slots, block_tables=t.block_tables, totals=t.totals,
                        request_tables=s["table"])
        if c["op"] == "window":
            return K.window_attention(s["q"], s["k"], s["v"], s["out"], s["start"], s["pos"], s["table"],
                                      window=c["window"], sinks=c["sinks"], max_query=s["most"],
                                      workspace=s["workspace"])
        return K.shared_prefix_attention(s["q"], s["k"], s["v"], s["out"], s["start"], s["pos"], s["table"],
                                         s["group_start"], s["prefix"], workspace=s["workspace"], **s["hints"])
    if c["op"] == "tables":
        return _plain_tables(s)
    if c["op"] == "window":
        return _plain_window(s)
    return _plain_prefix(s)


def _plain_tables(s: dict):
    c, req, W, cap = s["case"], s["request"].long(), s["case"]["max_blocks"], s["capacity"]
    S, dev = c["seqs"], req.device
    cached, new = s["cached"][req].long(), s["new"].long()
    cursor, n_free = s["cursor"].long(), s["free"].numel()
    wide = cached + new > W * PAGE
    n1 = torch.where(wide, 0, new)
    late = torch.cumsum(n1, 0) > cap
    n2 = torch.where(late, 0, n1)
    have = (cached + PAGE - 1) // PAGE
    need = (cached + n2 + PAGE - 1) // PAGE - have
    upto = torch.cumsum(need, 0)
    short = (cursor + upto > n_free) & (need > 0)
    n3 = torch.where(short, 0, n2)
    taken = torch.where(short, 0, need)
    start = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), torch.cumsum(n3, 0)])
    col = torch.arange(W, device=dev)[None, :]
    pick = (cursor + upto - need)[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < (have + taken)[:, None])
    rows = torch.where(col < have[:, None], s["table"][req].long(), -1)
    rows = torch.where(fresh, s["free"].long()[pick.clamp(0, n_free - 1)], rows)
    s["table"][req] = torch.where(fresh, rows.int(), s["table"][req])
    last = torch.full((1, W), -1, dtype=torch.long, device=dev)
    last[0, 0] = s["pad_block"]
    tables = torch.cat([rows, last])
    t = torch.arange(cap, device=dev)
    seq = torch.searchsorted(start[1:].contiguous(), t, right=True)  # S for the rows behind the last token
    real = seq < S
    at = seq.clamp(max=S - 1)
    pos = torch.where(real, cached[at] + t - start[at], 0)
    block = tables[seq, pos // PAGE]
    slots = torch.where(block >= 0, block * PAGE + pos % PAGE, -1)
    context = cached + n3
    status = 2 * wide.any().long() + 4 * late.any().long() + short.any().long()
    totals = torch.cat([start[-1:], cursor + taken.sum(), status[None], context.max()[None]])
    return dict(query_start=start.int(), context_len=context.int(), positions=pos.int(), token_seq=seq.int(),
                slots=slots, block_tables=tables.int(), totals=totals.int(), request_tables=s["table"])


def _attend(s: dict, kpos: torch.Tensor, seen) -> torch.Tensor:
    """Softmax attention in f32 of every sequence's tokens, padded to the most of one sequence, over its keys at
    positions kpos [S, L]; seen(query positions [S, M, 1], key positions [S, 1, L]) says which a token attends to."""
    q, start, table = s["q"], s["start"].long(), s["table"].long()
    T, H, KV, M = q.shape[0], q.shape[1], s["k"].shape[1], s["most"]
    i = torch.arange(M, device=q.device)[None, :]
    tok = start[:-1, None] + i
    real = tok < start[1:, None]
    tok = tok.clamp(max=T - 1)
    S, L = kpos.shape
    qp = torch.where(real, s["pos"].long()[tok], -1)[:, :, None]
    vis = seen(qp, kpos[:, None, :]) & (kpos >= 0)[:, None, :]
    page = (kpos.clamp(min=0) // PAGE).clamp(max=table.shape[1] - 1)
    block = torch.gather(table, 1, page).clamp(min=0)
    slot = kpos.clamp(min=0) % PAGE
    used = vis.any(1)[:, :, None, None]
    keys = torch.where(used, s["k"][block, :, slot].float(), 0.0)  # [S, L, KV, D]
    vals = torch.where(used, s["v"][block, :, slot].float(), 0.0)
    qq = q[tok].float().view(S, M, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(S, KV, M * (H // KV), D)
    score = torch.matmul(qq, keys.permute(0, 2, 3, 1).contiguous()) / math.sqrt(D)
    mask = vis[:, None, :, None, :].expand(S, KV, M, H // KV, L).reshape(S, KV, M * (H // KV), L)
    score = torch.where(mask, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    out = torch.matmul(w, vals.permute(0, 2, 1, 3).contiguous()) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    out = out.view(S, KV, M, H // KV, D).permute(0, 2, 1, 3, 4).reshape(S, M, H, D)
    return out[real].to(q.dtype)


def _plain_window(s: dict) -> torch.Tensor:
    c = s["case"]
    w, k, M = c["window"], c["sinks"], s["most"]
    dev = s["q"].device
    first = s["pos"].long()[s["start"].long()[:-1]]  # each sequence's first new token
    lo = torch.clamp(first - w + 1, min=0)[:, None]
    span = min(w + M - 1, s["longest"])
    near = lo + torch.arange(span, device=dev)[None, :]
    far = torch.arange(k, device=dev)[None, :].expand(lo.shape[0], k)
    kpos = torch.cat([torch.where(far < lo, far, -1), near], 1)
    return _attend(s, kpos, lambda qp, kp: (kp <= qp) & ((kp > qp - w) | (kp < k)))


def _plain_prefix(s: dict) -> torch.Tensor:
    kpos = torch.arange(s["longest"], device=s["q"].device)[None, :].expand(s["table"].shape[0], s["longest"])
    return _attend(s, kpos, lambda qp, kp: kp <= qp)


# ---- in 64 bits ----

def exact(case: dict, seed: int):
    """The attention outputs in float64, sequence by sequence; the tables are whole numbers and have none."""
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    H, KV = case["heads"], case["kv_heads"]
    start, pos, table = s["start"].tolist(), s["pos"].tolist(), s["table"].long()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i in range(case["seqs"]):
        a, b = start[i], start[i + 1]
        p = torch.tensor(pos[a:b], device=out.device)
        top = int(p.max()) + 1
        j = torch.arange(top, device=out.device)
        see = j[None, :] <= p[:, None]
        if case["op"] == "window":
            see &= (p[:, None] - j[None, :] < case["window"]) | (j[None, :] < case["sinks"])
        j = j[see.any(0)]
        see = see[:, j]
        blk = table[i, torch.div(j, PAGE, rounding_mode="floor")]
        key, val = s["k"][blk, :, j % PAGE].double(), s["v"][blk, :, j % PAGE].double()
        for h in range(H):
            kv = h // (H // KV)
            e = (s["q"][a:b, h].double() @ key[:, kv].T.contiguous()) * D ** -0.5
            e = torch.softmax(e.masked_fill(~see, -math.inf), 1)
            out[a:b, h] = e @ val[:, kv].contiguous()
    return out
