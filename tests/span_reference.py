"""Plain references of the step tables and of attention over spans of the paged cache, in Python and float64, with
the error bound of each output."""
from __future__ import annotations

import numpy as np

PAGE, D = 16, 128


def step_tables_reference(request, cached_len, new_len, request_tables, free_blocks, cursor, max_tokens, pad_block):
    """What step_tables writes, sequence by sequence. Returns a dict; `request_tables` in it is the updated copy."""
    tables = np.array(request_tables, np.int64)
    R, W = tables.shape
    S = len(new_len)
    request = np.arange(S) if request is None else np.asarray(request)
    cursor = min(max(cursor, 0), len(free_blocks))
    pages = lambda n: -(-n // PAGE)  # noqa: E731
    bits = 0
    rows, cached, new = [], [], []
    for s in range(S):
        r, n = int(request[s]), int(new_len[s])
        c = int(cached_len[r]) if 0 <= r < R else -1
        ok = 0 <= c <= W * PAGE and n >= 0 and list(request).count(r) == 1
        bits |= 0 if ok else 8
        if ok and c + n > W * PAGE:
            bits |= 2
            n = 0
        rows.append(r if ok else -1)
        cached.append(c if ok else 0)
        new.append(n if ok else 0)
    tokens = taken = 0  # of all sequences up to here, accepted or not
    out_new, at = [], []
    used = cursor
    for s in range(S):
        need = pages(cached[s] + new[s]) - pages(cached[s])
        tokens += new[s]
        taken += need
        if tokens > max_tokens:
            bits |= 4
            out_new.append(0)
        elif need and cursor + taken > len(free_blocks):
            bits |= 1
            out_new.append(0)
        else:
            out_new.append(new[s])
            at.append((s, used))
            used += need
    start = np.concatenate([[0], np.cumsum(out_new)]).astype(np.int64)
    step = np.full((S + 1, W), -1, np.int64)
    step[S, 0] = pad_block
    for s in range(S):
        if rows[s] >= 0:
            h = pages(cached[s])
            step[s, :h] = tables[rows[s], :h]
    for s, f in at:
        if rows[s] < 0:
            continue
        h, e = pages(cached[s]), pages(cached[s] + out_new[s])
        step[s, h:e] = tables[rows[s], h:e] = free_blocks[f:f + e - h]
    positions, token_seq = np.zeros(max_tokens, np.int64), np.full(max_tokens, S, np.int64)
    slots = np.full(max_tokens, pad_block * PAGE if pad_block >= 0 else -1, np.int64)
    for s in range(S):
        for i in range(out_new[s]):
            t, p = start[s] + i, cached[s] + i
            positions[t], token_seq[t] = p, s
            slots[t] = step[s, p // PAGE] * PAGE + p % PAGE if step[s, p // PAGE] >= 0 else -1
    context = np.array(cached, np.int64) + np.array(out_new, np.int64)
    totals = [start[-1], used, bits, max(context, default=0)]
    return dict(query_start=start, context_len=context, positions=positions, token_seq=token_seq, slots=slots,
                block_tables=step, totals=np.array(totals), request_tables=tables)


def attention_reference(q, k_pool, v_pool, tables, query_start, positions, sees, f16, scale=None):
    """softmax(scale q K^T) V per token in float64 over the keys j of its own table with sees(s, p, j).

    Returns (out, bound): the bound on |got - out| of a kernel with f32 scores and sums, and for f16 with weights and
    outputs rounded to f16. Its parts, for weights w (sum L = sum exp(s - max) >= 1) and values v:
      * a weight off by a factor 1 + e moves the output by e w |v - out|: e is half an f16 step (2^-11) for f16; the
        score's error, at most (128 + 2) 2^-24 sum |q k| scale for the products and sums and the scaling, and 2^-20
        for the exponentials of the weight and of the corrections (each 2^-22 and few);
      * a weight below the normal f16 range is off by half of 2^-24 at most, against L >= 1;
      * sums of n terms in f32: (n + 64) 2^-24 of sum w |v| and of |out|;
      * the output's own rounding, half a step of its value or of the smallest subnormal.
    """
    T, H = q.shape[:2]
    KV = k_pool.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, bound = np.zeros((T, H, D)), np.zeros((T, H, D))
    u = 2.0 ** -11 if f16 else 0.0
    for s in range(len(query_start) - 1):
        for t in range(query_start[s], query_start[s + 1]):
            p = int(positions[t])
            j = np.arange(min(p + 1, tables.shape[1] * PAGE))
            j = j[sees(s, p, j)] if j.size else j
            if not j.size:
                bound[t] = 0
                continue
            blk = tables[s, j // PAGE]
            K = np.where((blk >= 0)[:, None, None], k_pool[np.maximum(blk, 0), :, j % PAGE].astype(np.float64), 0)
            V = np.where((blk >= 0)[:, None, None], v_pool[np.maximum(blk, 0), :, j % PAGE].astype(np.float64), 0)
            for h in range(H):
                kk, vv, qq = K[:, h * KV // H], V[:, h * KV // H], q[t, h].astype(np.float64)
                e = kk @ qq * scale
                w = np.exp(e - e.max())
                L = w.sum()
                w = w / L
                o = w @ vv
                ds = 130 * 2.0 ** -24 * scale * (np.abs(kk) @ np.abs(qq)).max() + 2.0 ** -20
                away = np.abs(vv - o)
                n = j.size
                out[t, h] = o
                bound[t, h] = ((u + 2 * ds) * (w @ away) + (2.0 ** -25 / L * away.sum(0) if f16 else 0)
                               + (n + 64) * 2.0 ** -24 * (w @ np.abs(vv) + np.abs(o))
                               + (2.0 ** -11 * np.abs(o) + 2.0 ** -25 if f16 else 2.0 ** -24 * np.abs(o)))
    return out, bound
