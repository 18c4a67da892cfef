"""A cache and weights held in 4 bits, as cases that are measured.

Three operators of a serving step whose K/V pages and weights hold four bits a value (e2m1 codes in groups of 32, each
with a power-of-two scale byte). Sizes are the benchmark's and the tests': decode at batch 32 over 256 to 4096 tokens,
speculative verify at batch 64, 512-token prompt chunks, 2000 tokens on a 12,000-token context, 131,072-token contexts,
16 query and 8 kv heads of 128 (and the other head layouts of the tests), pages of 16 tokens; hidden 1024 and 2048,
vocabulary 151,936.

  append  qkv to q (norm and rotation, f16) and to the tokens' slots of the 4-bit pages.
  attn    causal attention of a ragged batch over 4-bit pages.
  gemv    activations times 4-bit weights, with the linear layers' epilogues.

Sequence lengths come from the case alone (its `lens`), values and page places from the seed. With ``own`` true ``run``
calls ``ember_amd.kernels``, else it computes the same in elementary torch operations.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE, D, GROUP = 16, 128, 32
PAGE_BYTES = 2 * PAGE * (D // 2 + D // GROUP)  # of one kv head: K codes, V codes, K scales, V scales
V_AT, KS_AT, VS_AT = PAGE * D // 2, PAGE * D, PAGE * D + PAGE * D // GROUP
LOWEST, HIGHEST = -23, 13  # exponents of a scale: every value that they allow is exact in f16

APPEND = dict(op="append", seqs=32, new=1, chunks=0, chunk=0, ctx_lo=256, ctx_hi=4095, heads=16, kv_heads=8, norm=True,
              bias=False, lens=1)
ATTN = dict(op="attn", seqs=1, new=1, ragged=False, ctx_lo=640, ctx_hi=640, heads=16, kv_heads=8, strided=False, lens=1)
GEMV = dict(op="gemv", rows=1, features=4096, inner=1024, epilogue="f16")


def listed() -> list:
    return [
        # A decode batch's append: one token of each of 32 sequences. All latency.
        dict(name="append_decode_b32", **APPEND),
        # A full card's step: 1000 decodes or verify runs, 12 of them a 512-token prompt chunk instead, biased projections.
        dict(name="append_mixed_b1000", **{**APPEND, **dict(seqs=1000, new=5, chunks=12, chunk=512, ctx_lo=64,
                                                            ctx_hi=130000, heads=32, bias=True, lens=2)}),
        # One user's chat turn: the smallest attention.
        dict(name="attn_decode_b1", **ATTN),
        # The benchmark's decode batch: 32 sequences of 256 to 4096 tokens.
        dict(name="attn_decode_b32", **{**ATTN, **dict(seqs=32, ctx_lo=256, ctx_hi=4095, lens=3)}),
        # Long documents: 8 sequences of up to 131,072 tokens, 4 query heads a kv head.
        dict(name="attn_decode_long_b8", **{**ATTN, **dict(seqs=8, ctx_lo=30000, ctx_hi=131000, heads=32, lens=4)}),
        # Speculative verify with 1 to 5 tokens a sequence, q a part of the projection's rows.
        dict(name="attn_verify_b64", **{**ATTN, **dict(seqs=64, new=5, ragged=True, ctx_lo=512, ctx_hi=4096,
                                                       strided=True, lens=5)}),
        # Prompt chunks of up to 512 tokens of 4 requests.
        dict(name="attn_prompt_4x512", **{**ATTN, **dict(seqs=4, new=512, ragged=True, ctx_lo=900, ctx_hi=3000, lens=6)}),
        # A long document's chunk: 2000 tokens on a 12,000-token context.
        dict(name="attn_prompt_2000", **{**ATTN, **dict(new=2000, ctx_lo=12000, ctx_hi=12000, lens=7)}),
        # One token's qkv projection: the smallest product.
        dict(name="gemv_qkv_b1", **GEMV),
        # Gate and up of 32 decodes, with the activation behind them.
        dict(name="gemv_gate_up_b32", **{**GEMV, **dict(rows=32, features=12288, inner=2048, epilogue="silu")}),
        # The vocabulary's logits of 8 decodes.
        dict(name="gemv_logits_b8", **{**GEMV, **dict(rows=8, features=151936, epilogue="f32")}),
        # A prompt chunk of 512 tokens through the down projection.
        dict(name="gemv_prompt_512", **{**GEMV, **dict(rows=512, features=2048, inner=6144, epilogue="f32")}),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(16, 8), (16, 8), (32, 8), (8, 8), (12, 4), (4, 2), (8, 1)]


def _draw_one(rng: random.Random) -> dict:
    op = rng.choice(["append", "attn", "attn", "gemv"])
    lens = rng.randrange(1 << 20)
    heads, kv = rng.choice(HEADS)
    if op == "gemv":
        rows = _log_int(rng, 1, 64) if rng.random() < 0.8 else _log_int(rng, 65, 512)
        epilogue = rng.choice(["f16", "f32", "silu"])
        return {**GEMV, **dict(rows=rows, features=2 * _log_int(rng, 8, 80000), inner=GROUP * _log_int(rng, 2, 192),
                               epilogue=epilogue)}
    if op == "append":
        seqs = _log_int(rng, 1, 1000)
        hi = _log_int(rng, 1, 130000)
        return {**APPEND, **dict(seqs=seqs, new=rng.choice([1, 1, 2, 5, 8]), chunks=rng.randint(0, min(seqs, 12)),
                                 chunk=_log_int(rng, 2, 512), ctx_lo=rng.randint(0, hi), ctx_hi=hi, heads=heads,
                                 kv_heads=kv, norm=rng.random() < 0.7, bias=rng.random() < 0.3, lens=lens)}
    kind = rng.choice(["decode", "decode", "verify", "prompt"])
    if kind == "prompt":
        seqs, new = _log_int(rng, 1, 6), _log_int(rng, 6, 2000)
    else:
        seqs, new = _log_int(rng, 1, 256), 1 if kind == "decode" else rng.randint(2, 8)
    hi = _log_int(rng, 1, 131000 if seqs <= 4 and kind == "decode" else 16384)
    return {**ATTN, **dict(seqs=seqs, new=new, ragged=rng.random() < 0.5, ctx_lo=rng.randint(0, hi), ctx_hi=hi,
                           heads=heads, kv_heads=kv, strided=rng.random() < 0.3, lens=lens)}


def draw(rng: random.Random) -> dict:
    top = {}
    for c in listed():
        w = work(c)
        for k in w:
            top[c["op"], k] = max(top.get((c["op"], k), 0), w[k])
    while True:
        c = _draw_one(rng)
        w = work(c)
        if all(w[k] <= top[c["op"], k] for k in w) and _memory(c) < 3e10:
            return c


# ---- lengths, from the case alone ----

def _lens(case: dict):
    """Per sequence the cached tokens and the new ones."""
    r = np.random.RandomState(case["lens"])
    S = case["seqs"]
    cached = r.randint(case["ctx_lo"], case["ctx_hi"] + 1, S)
    new = np.full(S, case["new"])
    if case["op"] == "append":
        new = r.randint(1, case["new"] + 1, S)
        new[r.permutation(S)[: case["chunks"]]] = case["chunk"] or case["new"]
    elif case["ragged"]:
        new = r.randint(1, case["new"] + 1, S)
    return cached, new


def work(case: dict) -> dict:
    if case["op"] == "gemv":
        M, N, K = case["rows"], case["features"], case["inner"]
        out = {"f16": 2 * N, "f32": 4 * N, "silu": N}[case["epilogue"]]
        return {"bytes": N * K // 2 + N * K // GROUP + 2 * M * K + M * out, "flops": 2 * M * N * K}
    cached, new = _lens(case)
    T, H, KV = int(new.sum()), case["heads"], case["kv_heads"]
    if case["op"] == "append":
        # qkv in; q, the values that K and V stand for, and the pages' codes and scales out
        return {"bytes": T * (2 * D * (2 * H + 4 * KV) + KV * PAGE_BYTES // PAGE), "flops": 0}
    pairs = int((new * cached + new * (new + 1) // 2).sum())
    return {"bytes": int((cached + new).sum()) * KV * PAGE_BYTES // PAGE + 4 * T * H * D, "flops": 4 * D * H * pairs}


def _memory(case: dict) -> float:
    """Bytes of the plain form's largest tensors."""
    if case["op"] == "gemv":
        return 16.0 * case["features"] * case["inner"]
    cached, new = _lens(case)
    if case["op"] == "append":
        return 64.0 * new.sum() * (case["heads"] + 2 * case["kv_heads"]) * D
    S, M, L = case["seqs"], int(new.max()), int((cached + new).max())
    return 4.0 * S * L * (4 * case["kv_heads"] * D + 3 * case["heads"] * M)


# ---- four bits in torch ----

def _encode(x: torch.Tensor):
    """Codes 0..15 like x [..., n] and scale bytes [..., n / 32], in x's own precision: the scale is the lowest power
    of two that leaves the group's largest value at 7 or less, a code the nearest of 0 .. 6, ties to the even code.
    Powers of two scale exactly, so 32 bits lose nothing here."""
    g = x.unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(m > 0.875, e - 2, e - 3).clamp(LOWEST, HIGHEST)
    e = torch.where(top == 0, LOWEST, e)
    y = g.abs() * torch.from_numpy(2.0 ** -np.arange(LOWEST, HIGHEST + 1.0)).to(x)[(e - LOWEST).long()][..., None]
    code = ((y > 0.25).byte() + (y >= 0.75).byte() + (y > 1.25).byte() + (y >= 1.75).byte() + (y > 2.5).byte()
            + (y >= 3.5).byte() + (y > 5.0).byte())
    return (code + 8 * torch.signbit(g).byte()).flatten(-2), (e + 127).byte()


def _decode(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The f32 values of codes 0..15 [..., n] with scale bytes [..., n / 32]."""
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    power = torch.from_numpy((2.0 ** (np.arange(256.0) - 127)).astype(np.float32)).to(code.device)
    return (lut[code.int()].unflatten(-1, (-1, GROUP)) * power[scale.int()][..., None]).flatten(-2)


def _nibbles(b: torch.Tensor) -> torch.Tensor:
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _bytes(code: torch.Tensor) -> torch.Tensor:
    return code[..., 0::2] | code[..., 1::2] << 4


def _to_pages(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Pages [n, KV, PAGE_BYTES] of K and V [n, KV, 16, 128]."""
    (kc, ks), (vc, vs) = _encode(k), _encode(v)
    kb = _bytes(kc).flatten(-2)
    vb = _bytes(vc).unflatten(-1, (16, 4)).unflatten(-3, (4, 4)).transpose(-3, -2).flatten(-4)  # [key / 4][dim / 8][key % 4][4]
    return torch.cat([kb, vb, ks.flatten(-2), vs.transpose(-2, -1).flatten(-2)], -1)


def _from_pages(p: torch.Tensor):
    """K and V [..., 16, 128] in f32 of pages [..., PAGE_BYTES]."""
    vb = p[..., V_AT:KS_AT].unflatten(-1, (4, 16, 4, 4)).transpose(-3, -2).flatten(-4, -3).flatten(-2)
    return (_decode(_nibbles(p[..., :V_AT].unflatten(-1, (PAGE, D // 2))), p[..., KS_AT:VS_AT].unflatten(-1, (PAGE, 4))),
            _decode(_nibbles(vb), p[..., VS_AT:].unflatten(-1, (4, PAGE)).transpose(-2, -1)))


# ---- inputs ----

def _channels(n: int, g: torch.Generator, dev) -> torch.Tensor:
    """Sizes of a head's channels: most alike, a few several times larger, as keys and activations have them."""
    return torch.exp(0.5 * torch.empty(n, device=dev).normal_(generator=g)).clamp(max=6.0)


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    normal = lambda *shape: torch.empty(shape, device=dev).normal_(generator=g)  # noqa: E731
    if case["op"] == "gemv":
        M, N, K = case["rows"], case["features"], case["inner"]
        code, scale = _encode(normal(N, K) * K ** -0.5 * _channels(N, g, dev)[:, None])
        s = dict(case=case, a=(normal(M, K) * _channels(K, g, dev)).half(), codes=_bytes(code), scales=scale)
        if own:
            from ember_amd import kernels as K4
            s["w"] = K4.gemv4_pack(s["codes"], s["scales"])
            s["c"] = torch.empty(M, N // 2 if case["epilogue"] == "silu" else N, device=dev,
                                 dtype=torch.float32 if case["epilogue"] == "f32" else torch.float16)
        return s
    r = np.random.RandomState(seed % (1 << 31))
    ints = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    cached, new = _lens(case)
    S, T, H, KV = case["seqs"], int(new.sum()), case["heads"], case["kv_heads"]
    ctx = cached + new
    W = int((ctx.max() + PAGE - 1) // PAGE) + 1
    col = np.arange(W)[None, :]
    live = col < ((ctx + PAGE - 1) // PAGE)[:, None]
    if case["op"] == "append":  # the pages that the step's tokens are in; the others' ids are never looked at
        live &= col >= (cached // PAGE)[:, None]
    total = int(live.sum())
    blocks = total + 7
    table = np.full((S, W), -1, np.int32)
    table[live] = r.permutation(blocks)[:total]
    start = np.concatenate([[0], np.cumsum(new)])
    pos = np.repeat(cached - start[:-1], new) + np.arange(T)
    pool = torch.empty(blocks, KV, PAGE_BYTES, dtype=torch.uint8, device=dev)
    k_size, v_size = _channels(D, g, dev), _channels(D, g, dev)
    for at in range(0, blocks, 4096):  # a part at a time: the values take 30 times the pages' memory
        n = min(4096, blocks - at)
        pool[at:at + n] = _to_pages((normal(n, KV, PAGE, D) * k_size).half().float(), (normal(n, KV, PAGE, D) * v_size).half().float())
    s = dict(case=case, pool=pool, table=ints(table), start=ints(start), pos=ints(pos), most=int(new.max()),
             longest=int(ctx.max()))
    if case["op"] == "append":
        width = (H + 2 * KV) * D
        s.update(qkv=(normal(T, width) * torch.exp(0.5 * normal(width))).half(), seq=ints(np.repeat(np.arange(S), new)),
                 inv_freq=torch.from_numpy((1e6 ** (-np.arange(0, D, 2) / D)).astype(np.float32)).to(dev),
                 q_norm=(1 + 0.3 * normal(D)) if case["norm"] else None,
                 k_norm=k_size.clone() if case["norm"] else None, bias=0.5 * normal(width) if case["bias"] else None)
        if own:
            e = lambda n: torch.empty(T, n, D, dtype=torch.float16, device=dev)  # noqa: E731
            s.update(q_out=e(H), k_out=e(KV), v_out=e(KV))
        return s
    row = (H + 2 * KV) * D if case["strided"] else H * D
    s["q"] = normal(T, row).half()[:, : H * D].view(T, H, D)
    if own:
        from ember_amd import kernels as K4
        s["out"] = torch.empty(T, H, D, dtype=torch.float16, device=dev)
        s["workspace"] = K4.kv4_workspace(T, S, n_heads=H, n_kv=KV, max_query=s["most"], max_context=s["longest"], device=dev)
    return s


# ---- the operators ----

def run(s: dict):
    c = s["case"]
    if own:
        from ember_amd import _lib
        from ember_amd import kernels as K
        if c["op"] == "append":
            K.kv4_append(s["qkv"], s["q_out"], s["pool"], s["pos"], s["seq"], s["table"], n_heads=c["heads"],
                         n_kv=c["kv_heads"], inv_freq_dev=s["inv_freq"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                         bias=s["bias"], k_out=s["k_out"], v_out=s["v_out"])
            return dict(q=s["q_out"], k=s["k_out"], v=s["v_out"], pages=s["pool"])
        if c["op"] == "attn":
            return K.kv4_attention(s["q"], s["pool"], s["out"], s["start"], s["pos"], s["table"], max_query=s["most"],
                                   max_context=s["longest"], workspace=s["workspace"])
        K.gemv4(s["a"], s["w"], s["c"], dict(f16=_lib.EPILOGUE_STORE_F16, f32=_lib.EPILOGUE_STORE_F32,
                                             silu=_lib.EPILOGUE_SILU_MUL)[c["epilogue"]], N=c["features"])
        return s["c"]
    if c["op"] == "append":
        return _plain_append(s)
    if c["op"] == "attn":
        return _plain_attn(s)
    y = torch.matmul(s["a"].float(), _decode(_nibbles(s["codes"]), s["scales"]).t())
    if c["epilogue"] == "f32":
        return y
    if c["epilogue"] == "silu":
        gate, up = y[:, 0::2], y[:, 1::2]
        y = gate / (1 + torch.exp(-gate)) * up
    return y.clamp(-65504, 65504).half()


def _plain_append(s: dict) -> dict:
    """In 32 bits, the sums of squares and the angles' sine and cosine in 64, as the f16 cache's append computes them."""
    c, pos = s["case"], s["pos"].long()
    T, H, KV = pos.numel(), c["heads"], c["kv_heads"]
    x = s["qkv"].float()
    if s["bias"] is not None:
        x = x + s["bias"]
    x = x.view(T, H + 2 * KV, D)
    qk, v = x[:, : H + KV], x[:, H + KV:]
    if s["q_norm"] is not None:
        w = torch.cat([s["q_norm"].expand(H, D), s["k_norm"].expand(KV, D)])
        qk = w * (qk * (1 / torch.sqrt(qk.double().square().mean(-1, keepdim=True) + 1e-6)).float())
    angle = (pos.float()[:, None] * s["inv_freq"]).double()[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    lo, hi = qk[..., : D // 2], qk[..., D // 2:]
    qk = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    (kc, ks), (vc, vs) = _encode(qk[:, H:]), _encode(v)
    block = s["table"].long()[s["seq"].long(), pos // PAGE][:, None, None]
    slot = (pos % PAGE)[:, None, None]
    head = torch.arange(KV, device=pos.device)[None, :, None]
    col, j = torch.arange(D // 2, device=pos.device), torch.arange(D // GROUP, device=pos.device)
    s["pool"][block, head, slot * (D // 2) + col] = _bytes(kc)
    s["pool"][block, head, V_AT + slot // 4 * 256 + col // 4 * 16 + slot % 4 * 4 + col % 4] = _bytes(vc)
    s["pool"][block, head, KS_AT + slot * 4 + j] = ks
    s["pool"][block, head, VS_AT + j * PAGE + slot] = vs
    return dict(q=qk[:, :H].half(), k=_decode(kc, ks).half(), v=_decode(vc, vs).half(), pages=s["pool"])


def _plain_attn(s: dict) -> torch.Tensor:
    """Softmax attention in f32 of every sequence's tokens, padded to the most of one sequence, over its keys."""
    q, start, table = s["q"], s["start"].long(), s["table"].long()
    T, H, KV, M, L = q.shape[0], q.shape[1], s["pool"].shape[1], s["most"], s["longest"]
    S, pages = table.shape[0], -(-L // PAGE)
    i = torch.arange(M, device=q.device)[None, :]
    tok = start[:-1, None] + i
    real = tok < start[1:, None]
    tok = tok.clamp(max=T - 1)
    top = torch.where(real, s["pos"].long()[tok], -1)[:, None, :, None, None]
    keys, vals = _from_pages(s["pool"][table[:, :pages].clamp(min=0)].transpose(1, 2))  # [S, KV, pages, 16, 128]
    keys, vals = (x.flatten(2, 3)[:, :, :L] for x in (keys, vals))
    qq = q[tok].float().view(S, M, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(S, KV, M * (H // KV), D)
    score = torch.matmul(qq, keys.transpose(-1, -2).contiguous()).view(S, KV, M, H // KV, L) / math.sqrt(D)
    score = torch.where(torch.arange(L, device=q.device) <= top, score, -math.inf)
    most = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(torch.isfinite(most), most, 0.0))
    out = torch.matmul(w.view(S, KV, -1, L), vals.contiguous()).view(S, KV, M, H // KV, D) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.permute(0, 2, 1, 3, 4).reshape(S, M, H, D)[real].half()


# ---- in 64 bits ----

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def _stood_for(x: torch.Tensor) -> torch.Tensor:
    """What x's groups of 32 come back as: the nearest level of the scale, of two as near the one of even number."""
    g = x.unflatten(-1, (-1, GROUP))
    powers = torch.from_numpy(2.0 ** np.arange(LOWEST, HIGHEST + 1.0)).to(x)
    at = torch.searchsorted(7 * powers, g.abs().amax(-1).contiguous()).clamp(max=powers.numel() - 1)  # the first that is enough
    unit = powers[at][..., None]
    far = torch.stack([(g.abs() / unit - level).abs() - (1e-13 if n % 2 == 0 else 0) for n, level in enumerate(LEVELS.tolist())])
    return (torch.sign(g) * torch.from_numpy(LEVELS).to(x)[far.argmin(0)] * unit).flatten(-2)


def _values(bytes_, scale):
    """Values in f64 of rows of packed codes: bytes [..., n / 2], scales [..., n / 32]."""
    level = torch.from_numpy(np.concatenate([LEVELS, -LEVELS])).to(bytes_.device)
    pair = torch.stack([level[(bytes_ % 16).long()], level[torch.div(bytes_, 16, rounding_mode="floor").long()]], -1)
    return pair.flatten(-2) * torch.exp2(scale.double() - 127).repeat_interleave(GROUP, -1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "gemv":
        y = torch.cat([s["a"].double() @ _values(s["codes"][i:i + 8192], s["scales"][i:i + 8192]).T.contiguous()
                       for i in range(0, case["features"], 8192)], 1)
        if case["epilogue"] == "silu":
            y = y[:, ::2] * torch.sigmoid(y[:, ::2]) * y[:, 1::2]
        return y
    H, KV = case["heads"], case["kv_heads"]
    pos = s["pos"]
    if case["op"] == "append":
        x = s["qkv"].double() + (0 if s["bias"] is None else s["bias"].double())
        heads = x.unflatten(1, (-1, D))
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), (pos.float()[:, None] * s["inv_freq"][None]).double())

        def rotated(y, w):
            if w is not None:
                y = y * w.double() * (y.square().sum(-1, keepdim=True) / D + 1e-6) ** -0.5
            z = torch.complex(y[..., :64].contiguous(), y[..., 64:].contiguous()) * turn[:, None]
            return torch.cat([z.real, z.imag], -1)

        return dict(q=rotated(heads[:, :H], s["q_norm"]), k=_stood_for(rotated(heads[:, H:H + KV], s["k_norm"])),
                    v=_stood_for(heads[:, H + KV:]), pages=None)
    start, table = s["start"].tolist(), s["table"].long()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i in range(case["seqs"]):
        a, b = start[i], start[i + 1]
        p = pos[a:b].long()
        top = int(p.max()) + 1
        pages = s["pool"][table[i, : -(-top // PAGE)]].transpose(0, 1)  # [KV, pages, bytes]
        see = torch.arange(top, device=p.device)[None, :] <= p[:, None]
        for kv in range(KV):
            byte = pages[kv]
            key = _values(byte[:, :V_AT].reshape(-1, D // 2), byte[:, KS_AT:VS_AT].reshape(-1, 4))[:top]
            vb = byte[:, V_AT:KS_AT].reshape(-1, 4, 16, 4, 4).permute(0, 1, 3, 2, 4).reshape(-1, D // 2)
            val = _values(vb, byte[:, VS_AT:].reshape(-1, 4, PAGE).permute(0, 2, 1).reshape(-1, 4))[:top]
            for h in range(kv * (H // KV), (kv + 1) * (H // KV)):
                e = (s["q"][a:b, h].double() @ key.T.contiguous()) * D ** -0.5
                out[a:b, h] = torch.softmax(e.masked_fill(~see, -math.inf), 1) @ val
    return out
