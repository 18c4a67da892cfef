"""Launchers of the gfx950 kernels through the C ABI, for torch tensors.

Mirrors the reference's launcher seam (src/backend/cuda/kernels.cuh:74-120):
``qk_norm_rope_store`` (-> ember_hip_kv_append), ``paged_attention``
(-> ember_hip_paged_decode), ``prefill_attention`` (-> ember_hip_prefill_attn),
plus ``copy_pages`` (copy-on-write). ``step_tables``, ``window_attention`` and
``shared_prefix_attention`` have no counterpart there: they take a step's integers
from the device, with no host plan. Nor have ``kv4_append``, ``kv4_attention``,
``mx_quantize``, ``gemv4_pack`` and ``gemv4``, for a cache and weights held in 4
bits, which do so too. Device tensors carry activations and pools;
the step's integer arrays are given as host arrays, checked here (every index a
kernel will follow is in range), then uploaded. Launches go to the current torch
stream unless ``stream`` is given.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib
from ._lib import BLOCK_SIZE, KV4_PAGE_BYTES, MAX_RUN, PREFILL_TILE, AttnArgs, CopyArgs, EmberError, PrefillArgs, QkvArgs, check

HEAD_DIM = 128


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.float16:
        return _lib.DTYPE_F16
    if t.dtype == torch.float32:
        return _lib.DTYPE_F32
    raise EmberError(f"unsupported dtype {t.dtype}")


def _stream_handle(stream) -> int:
    if stream is None:
        stream = torch.cuda.current_stream()
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _dev(t: torch.Tensor, name: str) -> int:
    if not t.is_cuda or not t.is_contiguous():
        raise EmberError(f"{name} must be a contiguous device tensor")
    return t.data_ptr()


def _opt(t: torch.Tensor | None, name: str) -> int | None:
    return None if t is None else _dev(t, name)


def _ints(a, device) -> torch.Tensor:
    return torch.as_tensor(np.ascontiguousarray(np.asarray(a, dtype=np.int32)), device=device)


@dataclass
class StepInts:
    """A step's integers on the host (the StepBatch fields the kernels read) and their device copies.

    positions [T], token_seq [T], block_tables [S, max_blocks].
    """

    positions: np.ndarray
    token_seq: np.ndarray
    block_tables: np.ndarray
    num_blocks: int  # blocks in each layer's pool (every table entry a kernel reads must be below it)

    def __post_init__(self):
        self.positions = np.ascontiguousarray(np.asarray(self.positions, dtype=np.int32).reshape(-1))
        self.token_seq = np.ascontiguousarray(np.asarray(self.token_seq, dtype=np.int32).reshape(-1))
        bt = np.asarray(self.block_tables, dtype=np.int32)
        self.block_tables = np.ascontiguousarray(bt.reshape(bt.shape[0], -1))
        T, S, W = self.positions.size, self.block_tables.shape[0], self.block_tables.shape[1]
        if self.token_seq.size != T:
            raise EmberError("positions and token_seq differ in length")
        if T and (self.token_seq.min() < 0 or self.token_seq.max() >= S):
            raise EmberError("token_seq names a sequence without a block table")
        if T and (self.positions.min() < 0 or self.positions.max() >= W * BLOCK_SIZE):
            raise EmberError("a position lies beyond its block table")
        for t in range(T):  # every page up to each token's position must be a pool block
            pages = self.block_tables[self.token_seq[t], : self.positions[t] // BLOCK_SIZE + 1]
            if pages.size and (pages.min() < 0 or pages.max() >= self.num_blocks):
                raise EmberError(f"token {t} reads a block outside the pool of {self.num_blocks}")
        self._dev = None

    @property
    def T(self) -> int:
        return int(self.positions.size)

    @property
    def max_blocks(self) -> int:
        return int(self.block_tables.shape[1])

    def device(self, device="cuda"):
        if self._dev is None:
            self._dev = (_ints(self.positions, device), _ints(self.token_seq, device), _ints(self.block_tables, device))
        return self._dev


def inv_freq(theta: float, head_dim: int = HEAD_DIM) -> np.ndarray:
    """Rotary frequencies in f32, as the reference computes them (cpu_backend.cpp:85-88)."""
    i = np.arange(head_dim // 2, dtype=np.float32)
    return (np.float32(1.0) / np.power(np.float32(theta), (2 * i) / np.float32(head_dim), dtype=np.float32)).astype(np.float32)


def qk_norm_rope_store(qkv, q_out, k_pool, v_pool, ints: StepInts, *, n_heads, n_kv, inv_freq_dev, q_norm=None,
                       k_norm=None, bias=None, eps=1e-6, stream=None):
    """QK-RMSNorm + RoPE + K/V page write for one layer (≙ cuda::qk_norm_rope_store)."""
    T = ints.T
    width = (n_heads + 2 * n_kv) * HEAD_DIM
    if qkv.numel() != T * width or q_out.numel() != T * n_heads * HEAD_DIM:
        raise EmberError("qkv / q_out sizes do not match the step")
    if k_pool.numel() < ints.num_blocks * n_kv * BLOCK_SIZE * HEAD_DIM or v_pool.numel() != k_pool.numel():
        raise EmberError("pools are smaller than num_blocks pages")
    pos, seq, tab = ints.device(qkv.device)
    a = QkvArgs()
    a.qkv, a.q_out = _dev(qkv, "qkv"), _dev(q_out, "q_out")
    a.k_cache, a.v_cache = _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")
    a.q_norm, a.k_norm, a.bias = _opt(q_norm, "q_norm"), _opt(k_norm, "k_norm"), _opt(bias, "bias")
    a.inv_freq = _dev(inv_freq_dev, "inv_freq")
    a.positions, a.token_seq, a.block_tables = pos.data_ptr(), seq.data_ptr(), tab.data_ptr()
    a.max_blocks, a.T, a.n_heads, a.n_kv, a.head_dim = ints.max_blocks, T, n_heads, n_kv, HEAD_DIM
    a.eps, a.num_blocks, a.dtype = eps, ints.num_blocks, _dtype_code(qkv)
    check(_lib.lib().ember_hip_kv_append(a, _stream_handle(stream)), "kv_append")


def decode_runs(ints: StepInts, token_list, max_run: int = MAX_RUN, group: int = 1):
    """Cuts a list of tokens into runs of consecutive tokens of one sequence, at most max_run each and at
    most 16 // group (a decode work-group holds at most 16 query rows: group heads x run tokens), the cap
    the C++ planner applies."""
    max_run = max(1, min(max_run, 16 // group))
    first, count = [], []
    i, tl = 0, list(token_list)
    while i < len(tl):
        j = i + 1
        while (j < len(tl) and j - i < max_run and tl[j] == tl[j - 1] + 1
               and ints.token_seq[tl[j]] == ints.token_seq[tl[i]] and ints.positions[tl[j]] == ints.positions[tl[j - 1]] + 1):
            j += 1
        first.append(i)
        count.append(j - i)
        i = j
    return np.asarray(first, np.int32), np.asarray(count, np.int32)


def work_list(run_ctx, split_len: int) -> np.ndarray:
    """(run, split) items, every full split first, then the partial last splits longest first
    (the order the C++ planner uses)."""
    full, partial = [], []
    for r, ctx in enumerate(int(c) for c in run_ctx):
        full += [(r, s) for s in range(ctx // split_len)]
        if ctx % split_len:
            partial.append((ctx % split_len, r, ctx // split_len))
    partial.sort(key=lambda x: -x[0])  # stable: equal sizes keep run order
    items = full + [(r, s) for _, r, s in partial]
    return np.asarray(items, np.int32).reshape(-1, 2)


def paged_attention(q, k_pool, v_pool, out, ints: StepInts, *, n_heads, n_kv, token_list=None, runs=None,
                    split_len=512, num_splits=None, scratch=None, use_work_list=False, merge_in_kernel=False,
                    work_desc=True, stream=None):
    """Paged decode attention (≙ cuda::paged_attention).

    token_list: tokens to process (None = all). runs: (run_first, run_count) over
    token_list positions, or None for one token per run. num_splits defaults to
    what the longest context needs at split_len keys per split. use_work_list:
    dispatch through a sorted (run, split) list instead of the dense grid.
    merge_in_kernel: merge the splits in the last work-group of each (run, kv
    head) instead of a second launch. work_desc: with the work list, also pass
    the per-item descriptors the C++ plan uploads (EmberAttnArgs::work_desc).
    """
    a, keep = _attn_args(q, k_pool, v_pool, out, ints, n_heads=n_heads, n_kv=n_kv, token_list=token_list, runs=runs,
                         split_len=split_len, num_splits=num_splits, scratch=scratch, use_work_list=use_work_list,
                         merge_in_kernel=merge_in_kernel, work_desc=work_desc)
    if a is None:
        return keep
    check(_lib.lib().ember_hip_paged_decode(a, _stream_handle(stream)), "paged_decode")
    return keep  # the caller keeps the uploads alive until the stream has run


def decode_step(qkv, k_pool, v_pool, out, ints: StepInts, *, n_heads, n_kv, inv_freq_dev, q_norm=None, k_norm=None,
                bias=None, eps=1e-6, runs=None, split_len=512, num_splits=None, use_work_list=False,
                merge_in_kernel=False, work_desc=True, stream=None):
    """Append + attention in one launch (ember_hip_decode_step); every token of the step is listed, each
    sequence's tokens forming one run of consecutive positions."""
    T = ints.T
    width = (n_heads + 2 * n_kv) * HEAD_DIM
    if qkv.numel() != T * width:
        raise EmberError("qkv does not match the step")
    a, keep = _attn_args(None, k_pool, v_pool, out, ints, n_heads=n_heads, n_kv=n_kv, token_list=None, runs=runs,
                         split_len=split_len, num_splits=num_splits, scratch=None, use_work_list=use_work_list,
                         merge_in_kernel=merge_in_kernel, work_desc=work_desc, dtype_of=qkv)
    seqs = ints.token_seq.tolist()
    if runs is None and len(set(seqs)) != len(seqs):
        raise EmberError("a sequence with several tokens needs them as one run")
    if runs is not None:  # one run per sequence, consecutive positions (the kernel relies on both)
        seen = set()
        for f, c in zip(*runs):
            s = int(ints.token_seq[f])
            if s in seen or np.any(np.diff(ints.positions[f:f + c]) != 1):
                raise EmberError("each sequence's tokens must form one run of consecutive positions")
            seen.add(s)
    pos, seq, tab = ints.device(qkv.device)
    qa = QkvArgs()
    qa.qkv, qa.q_out = _dev(qkv, "qkv"), None
    qa.k_cache, qa.v_cache = a.k_cache, a.v_cache
    qa.q_norm, qa.k_norm, qa.bias = _opt(q_norm, "q_norm"), _opt(k_norm, "k_norm"), _opt(bias, "bias")
    qa.inv_freq = _dev(inv_freq_dev, "inv_freq")
    qa.positions, qa.token_seq, qa.block_tables = pos.data_ptr(), seq.data_ptr(), tab.data_ptr()
    qa.max_blocks, qa.T, qa.n_heads, qa.n_kv, qa.head_dim = ints.max_blocks, T, n_heads, n_kv, HEAD_DIM
    qa.eps, qa.num_blocks, qa.dtype = eps, ints.num_blocks, _dtype_code(qkv)
    check(_lib.lib().ember_hip_decode_step(qa, a, _stream_handle(stream)), "decode_step")
    return keep


def _attn_args(q, k_pool, v_pool, out, ints: StepInts, *, n_heads, n_kv, token_list, runs, split_len, num_splits,
               scratch, use_work_list, merge_in_kernel, work_desc=True, dtype_of=None):
    tl = np.arange(ints.T, dtype=np.int32) if token_list is None else np.asarray(token_list, np.int32)
    n = int(tl.size)
    if n == 0:
        return None, []
    if tl.min() < 0 or tl.max() >= ints.T:
        raise EmberError("token_list names a token outside the step")
    if (q is not None and q.numel() < ints.T * n_heads * HEAD_DIM) or out.numel() < ints.T * n_heads * HEAD_DIM:
        raise EmberError("q / out are smaller than the step")
    if k_pool.numel() < ints.num_blocks * n_kv * BLOCK_SIZE * HEAD_DIM:
        raise EmberError("pools are smaller than num_blocks pages")
    ctx = int(ints.positions[tl].max()) + 1
    if num_splits is None:
        num_splits = max(1, math.ceil(ctx / split_len))
    if num_splits * split_len < ctx:
        raise EmberError("num_splits x split_len does not cover the context")
    dev = k_pool.device
    pos, seq, tab = ints.device(dev)
    tl_dev = _ints(tl, dev)
    a = AttnArgs()
    a.token_index = tl_dev.data_ptr()
    a.q = None if q is None else _dev(q, "q")
    a.k_cache, a.v_cache = _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")
    a.positions, a.token_seq, a.block_tables = pos.data_ptr(), seq.data_ptr(), tab.data_ptr()
    a.max_blocks, a.T, a.n_heads, a.n_kv, a.head_dim = ints.max_blocks, n, n_heads, n_kv, HEAD_DIM
    a.scale = 1.0 / math.sqrt(HEAD_DIM)
    a.out = _dev(out, "out")
    a.num_splits, a.split_len = num_splits, split_len
    keep = [tl_dev]
    if num_splits > 1:
        need = n * n_heads * num_splits
        if scratch is None:
            scratch = (torch.empty(need * HEAD_DIM, dtype=torch.float32, device=dev),
                       torch.empty(need * 2, dtype=torch.float32, device=dev))
        if scratch[0].numel() < need * HEAD_DIM or scratch[1].numel() < need * 2:
            raise EmberError("split scratch too small")
        a.part_acc, a.part_ml = _dev(scratch[0], "part_acc"), _dev(scratch[1], "part_ml")
        keep.append(scratch)
    a.num_blocks, a.dtype = ints.num_blocks, _dtype_code(q if q is not None else dtype_of)
    if runs is not None:
        rf, rc = (np.asarray(x, np.int32) for x in runs)
        if rf.size != rc.size or rc.min() < 1 or rc.max() > MAX_RUN or rf.min() < 0 or (rf + rc).max() > n:
            raise EmberError("malformed runs")
        for f, c in zip(rf, rc):  # one sequence per run
            if len(set(ints.token_seq[tl[f:f + c]].tolist())) != 1:
                raise EmberError("a run spans two sequences")
        rf_dev, rc_dev = _ints(rf, dev), _ints(rc, dev)
        keep += [rf_dev, rc_dev]
        a.run_first, a.run_count, a.num_runs, a.max_run = rf_dev.data_ptr(), rc_dev.data_ptr(), int(rf.size), int(rc.max())
        run_ctx = [int(ints.positions[tl[f:f + c]].max()) + 1 for f, c in zip(rf, rc)]
    else:
        rf, rc = np.arange(n, dtype=np.int32), np.ones(n, np.int32)
        run_ctx = [int(ints.positions[t]) + 1 for t in tl]
    if use_work_list:
        items = work_list(run_ctx, split_len)
        if items.size and items[:, 1].max() >= num_splits:
            raise EmberError("num_splits is too small for the work list")
        w_dev = _ints(items.reshape(-1), dev)
        keep.append(w_dev)
        a.work, a.num_work = w_dev.data_ptr(), int(items.shape[0])
        if work_desc:
            desc = np.full((items.shape[0], 16), -1, np.int32)
            for i, (r, sp) in enumerate(items.tolist()):
                toks = tl[rf[r]:rf[r] + rc[r]]
                pos = ints.positions[toks]
                seq = int(ints.token_seq[toks[0]])
                counting = (np.diff(toks) == 1).all() and (np.diff(pos) == 1).all()
                desc[i, :8] = (r, sp, rf[r], rc[r], seq, pos.min(), pos.max(), toks[0] if counting else -1)
                p0 = sp * split_len // BLOCK_SIZE
                last = min(int(pos.max()) + 1, (sp + 1) * split_len) - 1
                for j in range(8):
                    if p0 + j <= last // BLOCK_SIZE:
                        desc[i, 8 + j] = ints.block_tables[seq, p0 + j]
            d_dev = _ints(desc.reshape(-1), dev)
            keep.append(d_dev)
            a.work_desc = d_dev.data_ptr()
    if merge_in_kernel:
        counters = torch.zeros(len(run_ctx) * n_kv, dtype=torch.int32, device=dev)
        keep.append(counters)
        a.merge_counters = counters.data_ptr()
    return a, keep


def prefill_attention(q, k_pool, v_pool, out, ints: StepInts, *, n_heads, n_kv, tiles, stream=None,
                      heads_per_group=0):
    """Causal prefill attention of query tiles on MFMA (≙ cuda::prefill_attention).

    tiles: (start, end, seq) triples, each up to PREFILL_TILE consecutive tokens start..end-1 of
    sequence seq; every token attends to its sequence's keys 0..its position, which must already be in
    the pools. f16 only. heads_per_group: 0 (the launcher's choice), 1 or 2 (even G): the same bits.
    """
    if not tiles:
        return []
    t = np.asarray(tiles, np.int32).reshape(-1, 3)
    if (t[:, 1] <= t[:, 0]).any() or (t[:, 1] - t[:, 0] > PREFILL_TILE).any() or t[:, 0].min() < 0 \
            or t[:, 1].max() > ints.T:
        raise EmberError("malformed tiles")
    for s0, e0, sq in t.tolist():
        if (ints.token_seq[s0:e0] != sq).any():
            raise EmberError("a tile spans tokens of another sequence")
    if q.numel() < ints.T * n_heads * HEAD_DIM or out.numel() < ints.T * n_heads * HEAD_DIM:
        raise EmberError("q / out are smaller than the step")
    if k_pool.numel() < ints.num_blocks * n_kv * BLOCK_SIZE * HEAD_DIM:
        raise EmberError("pools are smaller than num_blocks pages")
    dev = k_pool.device
    pos, seq, tab = ints.device(dev)
    ts, te, tq = (_ints(np.ascontiguousarray(t[:, i]), dev) for i in range(3))
    a = PrefillArgs()
    a.q, a.k_cache, a.v_cache = _dev(q, "q"), _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")
    a.tile_start, a.tile_end, a.tile_seq = ts.data_ptr(), te.data_ptr(), tq.data_ptr()
    a.positions, a.block_tables = pos.data_ptr(), tab.data_ptr()
    a.num_tiles, a.max_blocks, a.n_heads, a.n_kv, a.head_dim = int(t.shape[0]), ints.max_blocks, n_heads, n_kv, HEAD_DIM
    a.scale = 1.0 / math.sqrt(HEAD_DIM)
    a.out = _dev(out, "out")
    a.num_blocks, a.dtype = ints.num_blocks, _dtype_code(q)
    a.heads_per_group = heads_per_group
    check(_lib.lib().ember_hip_prefill_attn(a, _stream_handle(stream)), "prefill_attn")
    return [ts, te, tq]


def copy_pages(k_pool, v_pool, src, dst, *, n_layers, layer_stride, n_kv, num_blocks, stream=None):
    """Copies whole pages src[i] -> dst[i] over every layer (the device half of copy-on-write)."""
    s, d = np.asarray(src, np.int32), np.asarray(dst, np.int32)
    if s.size != d.size:
        raise EmberError("src / dst differ in length")
    if s.size == 0:
        return
    if min(s.min(), d.min()) < 0 or max(s.max(), d.max()) >= num_blocks:
        raise EmberError("a page pair lies outside the pool")
    if k_pool.numel() < n_layers * layer_stride:
        raise EmberError("pools are smaller than n_layers x layer_stride")
    dev = k_pool.device
    sd, dd = _ints(s, dev), _ints(d, dev)
    a = CopyArgs()
    a.k_cache, a.v_cache = _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")
    a.src_blocks, a.dst_blocks, a.n = sd.data_ptr(), dd.data_ptr(), int(s.size)
    a.n_layers, a.layer_stride, a.n_kv, a.head_dim = n_layers, layer_stride, n_kv, HEAD_DIM
    a.num_blocks, a.dtype = num_blocks, _dtype_code(k_pool)
    check(_lib.lib().ember_hip_copy_pages(a, _stream_handle(stream)), "copy_pages")
    return (sd, dd)


def gemv_workspace(M: int, N: int, K: int, device="cuda"):
    """A zeroed workspace for gemv at this shape (uint8 tensor), or None when the shape does not split K."""
    n = int(_lib.lib().ember_hip_gemv_workspace_bytes(M, N, K))
    return torch.zeros(n, dtype=torch.uint8, device=device) if n > 0 else None


def gemv_pack(w, stream=None):
    """W (f16 [N, K]) laid out for gemv(..., packed=True): a flat f16 device tensor (N rounded up to 16 rows)."""
    if w.dtype != torch.float16 or w.dim() != 2:
        raise EmberError("gemv_pack: w must be f16 [N, K]")
    N, K = w.shape
    n = int(_lib.lib().ember_hip_gemv_packed_bytes(N, K))
    if n <= 0:
        raise EmberError(f"gemv_pack: K must be a positive multiple of 32 (got {K})")
    out = torch.empty(n // 2, dtype=torch.float16, device=w.device)
    check(_lib.lib().ember_hip_gemv_pack(_dev(w, "w"), N, K, out.data_ptr(), _stream_handle(stream)), "gemv_pack")
    return out


def gemv(a, w, c, epilogue: int, stream=None, workspace=None, packed=None):
    """C = A . W^T for decode-sized batches (≙ cuda::gemm with GemmKernel::gemv_tc, k_gemm.cu:302-425).

    a: f16 [M, K] (M <= 64, K a multiple of 32); w: f16 [N, K]; c: per epilogue, f16 [M, N] (store_f16),
    f32 [M, N] (store_f32; add_f32 adds into it) or f16 [M, N / 2] (silu_mul, W rows interleaving gate and up).
    workspace: None, or a zeroed device tensor of at least gemv_workspace's size, which lets a shape with few
    output features split K over more work-groups (not shared by launches that overlap in time).
    packed: None, or gemv_pack(w): the kernel then reads W from that layout (the same bits); w still gives N, K.
    """
    if a.dtype != torch.float16 or w.dtype != torch.float16 or a.dim() != 2 or w.dim() != 2 or a.shape[1] != w.shape[1]:
        raise EmberError("gemv: a [M, K] and w [N, K] must be f16 with the same K")
    M, K = a.shape
    N = w.shape[0]
    cols = N // 2 if epilogue == _lib.EPILOGUE_SILU_MUL else N
    want = torch.float32 if epilogue in (_lib.EPILOGUE_STORE_F32, _lib.EPILOGUE_ADD_F32) else torch.float16
    if c.dtype != want or tuple(c.shape) != (M, cols):
        raise EmberError(f"gemv: c must be {want} [{M}, {cols}]")
    g = _lib.GemvArgs()
    g.A, g.lda, g.W, g.M, g.N, g.K = _dev(a, "a"), K, _dev(w, "w"), M, N, K
    g.C, g.ldc, g.epilogue = _dev(c, "c"), cols, epilogue
    if workspace is not None:
        g.workspace, g.workspace_bytes = _dev(workspace, "workspace"), workspace.numel() * workspace.element_size()
    if packed is not None:
        g.W, g.w_packed = _dev(packed, "packed w"), 1
    check(_lib.lib().ember_hip_gemv(g, _stream_handle(stream)), "gemv")


def rmsnorm_rows(x, w, out, eps: float, rows=None, stream=None):
    """out[r] = rmsnorm(x[rows[r] if rows else r]) * w as f16 (≙ cuda::rmsnorm_rows, kernels.cuh:70-72)."""
    if x.dtype != torch.float32 or w.dtype != torch.float32 or out.dtype != torch.float16:
        raise EmberError("rmsnorm_rows: x and w f32, out f16")
    hidden = x.shape[-1]
    R = out.shape[0]
    keep = []
    n = _lib.NormArgs()
    n.x, n.w, n.out, n.R, n.hidden, n.eps = _dev(x, "x"), _dev(w, "w"), _dev(out, "out"), R, hidden, eps
    if rows is not None:
        r = _ints(np.asarray(rows, np.int32), x.device)
        keep.append(r)
        n.rows = r.data_ptr()
    check(_lib.lib().ember_hip_rmsnorm_rows(n, _stream_handle(stream)), "rmsnorm_rows")
    return keep


# The calls below run once per layer or step around kernels of a few microseconds, so what they check, they check with
# few Python operations.

def _launch(fn, args, dev: int, stream, what: str) -> None:
    """fn(args, stream) on device `dev`: on `stream`, or on torch's current stream of that device."""
    if stream is None:
        handle = torch._C._cuda_getCurrentRawStream(dev)
    else:
        handle = stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)
    if dev == torch.cuda.current_device():
        code = fn(args, handle)
    else:
        with torch.cuda.device(dev):
            code = fn(args, handle)
    if code:
        check(code, what)


def _new_on(device, stream, make, *shape):
    """make(shape) in uint8 (torch.empty or torch.zeros) for a launch on `stream`: its memory is not one that another
    stream still uses, and is written in that stream's order."""
    if stream is None:
        return make(shape, dtype=torch.uint8, device=device)
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    with torch.cuda.stream(stream):
        return make(shape, dtype=torch.uint8, device=device)


def _refuse(tensors: dict, dev: int, dtype) -> None:
    """Names the first of these tensors that is not a contiguous `dtype` tensor on device `dev`."""
    for name, t in tensors.items():
        if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
            raise EmberError(f"{name} must be a contiguous {dtype} tensor on cuda:{dev}")


class StepTables:
    """A step's integers on the device, as step_tables writes them: query_start [S + 1], context_len [S],
    positions / token_seq / slots [max_tokens], block_tables [S + 1, max_blocks], totals [4] (tokens, entries of
    the free list taken by now, STEP_* bits, longest context)."""

    def __init__(self, S: int, max_tokens: int, max_blocks: int, device="cuda"):
        e = lambda *shape, dtype=torch.int32: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
        self.S, self.max_tokens, self.max_blocks = S, max_tokens, max_blocks
        self.query_start, self.context_len = e(S + 1), e(S)
        self.positions, self.token_seq, self.slots = e(max_tokens), e(max_tokens), e(max_tokens, dtype=torch.int64)
        self.block_tables, self.totals = e(S + 1, max_blocks), e(4)
        if not self.totals.is_cuda:
            raise EmberError("StepTables live on the device")
        a = self._args = _lib.StepTablesArgs()  # what no call changes
        a.S, a.max_tokens, a.max_blocks = S, max_tokens, max_blocks
        a.query_start, a.context_len = self.query_start.data_ptr(), self.context_len.data_ptr()
        a.positions, a.token_seq, a.slots = self.positions.data_ptr(), self.token_seq.data_ptr(), self.slots.data_ptr()
        a.block_tables, a.totals = self.block_tables.data_ptr(), self.totals.data_ptr()


def step_tables(out: StepTables, request_tables, cached_len, new_len, free_blocks, *, request=None, free_cursor=None,
                pad_block: int = -1, stream=None) -> StepTables:
    """The integers of a step from its requests' lengths, in one launch (ember_hip_step_tables).

    request_tables [R, max_blocks]: each request's pages; the pages the step takes from free_blocks (from entry
    free_cursor[0] on) are written behind them. cached_len [R]; new_len [S]; request [S] (None: rows 0..S-1).
    All int32 on out's device. Nothing is checked on the host that would need the device's values: totals[2]
    says which sequences got no tokens and why.
    """
    dev, i32 = out.totals.get_device(), torch.int32
    for t in (request_tables, cached_len, new_len, free_blocks):
        if t.dtype is not i32 or t.get_device() != dev or not t.is_contiguous():
            _refuse(dict(request_tables=request_tables, cached_len=cached_len, new_len=new_len, free_blocks=free_blocks), dev, i32)
    R = len(request_tables)
    if request_tables.shape != (R, out.max_blocks) or cached_len.shape != (R,) or new_len.shape != (out.S,) \
            or free_blocks.dim() != 1:
        raise EmberError(f"request_tables, cached_len, new_len and free_blocks must be [R, {out.max_blocks}], [R], "
                         f"[{out.S}] and a list")
    a = out._args
    a.request_tables, a.cached_len = request_tables.data_ptr(), cached_len.data_ptr()
    a.new_len, a.free_blocks = new_len.data_ptr(), free_blocks.data_ptr()
    a.request = a.free_cursor = None
    if request is not None:
        _refuse(dict(request=request), dev, i32)
        if request.shape != new_len.shape:
            raise EmberError("request must name a row for each new_len")
        a.request = request.data_ptr()
    if free_cursor is not None:
        _refuse(dict(free_cursor=free_cursor), dev, i32)
        if free_cursor.numel() != 1:
            raise EmberError("free_cursor must be one number")
        a.free_cursor = free_cursor.data_ptr()
    if not -1 <= pad_block <= 0x7FFFFFFF:
        raise EmberError(f"pad_block is a page or -1 (got {pad_block})")
    a.R, a.n_free, a.pad_block = R, len(free_blocks), pad_block
    _launch(_lib.lib().ember_hip_step_tables, a, dev, stream, "step_tables")
    return out


def _check_kv4_pool(pool, dev: int) -> None:
    """A pool of 4-bit pages on device `dev`."""
    if pool.dtype is not torch.uint8 or pool.get_device() != dev or not pool.is_contiguous():
        _refuse(dict(pool=pool), dev, torch.uint8)
    shape = pool.shape
    if len(shape) != 3 or shape[2] != KV4_PAGE_BYTES:
        raise EmberError(f"pool must be [num_blocks, n_kv, {KV4_PAGE_BYTES}]")


def _ragged_batch(q, k_pool, v_pool, out, query_start, positions, block_tables, max_query, scale, workspace):
    """Checks a ragged batch and returns its device and the fields of an EmberRaggedBatch, in order: q [T, n_heads, 128]
    (any token stride), pools [num_blocks, n_kv, 16, 128]; k_pool [num_blocks, n_kv, KV4_PAGE_BYTES] of 4-bit pages where
    v_pool is None."""
    dev, dtype, i32 = q.get_device(), q.dtype, torch.int32
    if dev < 0 or not (dtype is torch.float16 or dtype is torch.float32):
        raise EmberError(f"q must be an f16 or f32 device tensor (got {dtype} on {q.device})")
    for t in (k_pool, v_pool, out) if v_pool is not None else (out,):
        if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
            _refuse(dict(k_pool=k_pool, v_pool=v_pool, out=out) if v_pool is not None else dict(out=out), dev, dtype)
    for t in (query_start, positions, block_tables):
        if t.dtype is not i32 or t.get_device() != dev or not t.is_contiguous():
            _refuse(dict(query_start=query_start, positions=positions, block_tables=block_tables), dev, i32)
    shape, pool, stride = q.shape, k_pool.shape, q.stride()
    if len(shape) != 3 or shape[2] != HEAD_DIM or stride[2] != 1 or stride[1] != HEAD_DIM:
        raise EmberError("q must be [T, n_heads, 128] with each token's heads contiguous")
    if v_pool is None:
        _check_kv4_pool(k_pool, dev)
        if out.shape != shape:
            raise EmberError("out must be shaped like q")
    elif len(pool) != 4 or pool[2] != BLOCK_SIZE or pool[3] != HEAD_DIM or v_pool.shape != pool or out.shape != shape:
        raise EmberError("pools must be [num_blocks, n_kv, 16, 128] alike, and out shaped like q")
    T, H, _ = shape
    S = query_start.numel() - 1
    table = block_tables.shape
    if S < 0 or positions.numel() < T or len(table) != 2 or table[0] < S:
        raise EmberError("query_start must be [S + 1], positions hold every token, block_tables be [S, max_blocks] (or more rows)")
    ws = ws_bytes = 0
    if workspace is not None:
        if workspace.get_device() != dev or not workspace.is_contiguous():
            raise EmberError(f"workspace must be a contiguous tensor on cuda:{dev}")
        ws, ws_bytes = workspace.data_ptr(), workspace.nbytes
    return dev, (q.data_ptr(), k_pool.data_ptr(), 0 if v_pool is None else v_pool.data_ptr(), out.data_ptr(), query_start.data_ptr(),
                 positions.data_ptr(), block_tables.data_ptr(), stride[0] if T > 1 else H * HEAD_DIM, T, S, table[1], H,
                 pool[1], HEAD_DIM, pool[0], _lib.DTYPE_F16 if dtype is torch.float16 else _lib.DTYPE_F32,
                 HEAD_DIM ** -0.5 if scale is None else scale, (T or 1) if max_query is None else max_query, ws, ws_bytes)


def _batch_sizes(T, S, n_heads, n_kv, max_query, dtype, max_blocks):
    """The fields of an EmberRaggedBatch of which only the sizes count."""
    return (0, 0, 0, 0, 0, 0, 0, n_heads * HEAD_DIM, T, S, 1 << 26 if max_blocks is None else max_blocks, n_heads, n_kv,
            HEAD_DIM, 1, _lib.DTYPE_F16 if dtype == torch.float16 else _lib.DTYPE_F32, 1.0,
            (T or 1) if max_query is None else max_query, 0, 0)


def _workspace_bytes(size, args) -> int:
    n = int(size(args))
    if n == 0 and _lib.last_error():  # sizes that no call takes
        raise EmberError(_lib.last_error())
    return n


def _workspace(size, args, dtype, device):
    """A workspace of size(args) bytes, or None for 0 of them."""
    if not (dtype is torch.float16 or dtype is torch.float32):
        raise EmberError(f"dtype must be f16 or f32 (got {dtype})")
    n = _workspace_bytes(size, args)
    return torch.empty(n, dtype=torch.uint8, device=device) if n > 0 else None


def _check_window(window: int, sinks: int) -> None:
    if not (0 < window <= 0x7FFFFFFF and 0 <= sinks <= 0x7FFFFFFF):
        raise EmberError(f"window must be 1 .. 2^31 - 1 and sinks 0 .. 2^31 - 1 (got {window}, {sinks})")


def window_workspace(T: int, S: int, *, n_heads, n_kv, window, sinks=0, max_query=None, dtype=torch.float16,
                     max_blocks=None, device="cuda"):
    """A workspace for window_attention of batches of these sizes and smaller ones (padded or not), or None when no such
    call splits its keys."""
    _check_window(window, sinks)
    a = _lib.WindowAttnArgs(*_batch_sizes(T, S, n_heads, n_kv, max_query, dtype, max_blocks), window, sinks)
    return _workspace(_lib.lib().ember_hip_window_workspace_bytes, a, dtype, device)


def window_attention(q, k_pool, v_pool, out, query_start, positions, block_tables, *, window: int, sinks: int = 0,
                     max_query=None, scale=None, workspace=None, stream=None):
    """Attention of each token to itself, the window - 1 tokens before it and its sequence's first `sinks` tokens
    (ember_hip_window_attn); returns out.

    q [T, n_heads, 128] (a part of wider rows is fine), out the same, contiguous; pools [num_blocks, n_kv, 16, 128];
    query_start [S + 1], positions [T] and block_tables [S, max_blocks] int32 on the device, as step_tables writes
    them. Pages that no token of the step attends to are not read and may have been freed. Rows of q past
    query_start[S] are left alone. max_query: the most tokens of one sequence (None: T); workspace: of
    window_workspace, not shared by calls that overlap in time (None: no splits).
    """
    _check_window(window, sinks)
    dev, batch = _ragged_batch(q, k_pool, v_pool, out, query_start, positions, block_tables, max_query, scale, workspace)
    _launch(_lib.lib().ember_hip_window_attn, _lib.WindowAttnArgs(*batch, window, sinks), dev, stream, "window_attn")
    return out


def _prefix_sizes(T, n_groups, max_group, max_prefix, max_own, max_blocks):
    far = min(max_blocks * BLOCK_SIZE, 0x7FFFFFFF)
    return (n_groups, (T or 1) if max_group is None else max_group, far if max_prefix is None else max_prefix,
            far if max_own is None else max_own)


def shared_prefix_workspace(T: int, S: int, n_groups: int, *, n_heads, n_kv, max_query=None, max_group=None,
                            max_prefix=None, max_own=None, dtype=torch.float16, max_blocks=None, device="cuda"):
    """A workspace for shared_prefix_attention of batches of these sizes."""
    batch = _batch_sizes(T, S, n_heads, n_kv, max_query, dtype, max_blocks)
    a = _lib.PrefixAttnArgs(*batch, 0, 0, *_prefix_sizes(T, n_groups, max_group, max_prefix, max_own, batch[10]))
    return _workspace(_lib.lib().ember_hip_shared_prefix_workspace_bytes, a, dtype, device)


def shared_prefix_attention(q, k_pool, v_pool, out, query_start, positions, block_tables, group_start, prefix_len, *,
                            max_query=None, max_group=None, max_prefix=None, max_own=None, scale=None, workspace=None,
                            stream=None):
    """Causal attention of groups of sequences that share a cached prefix, read for the group and not for each sequence
    (ember_hip_shared_prefix_attn); returns out.

    As window_attention, and: group_start [n_groups + 1], group g being sequences group_start[g] ..
    group_start[g + 1] - 1; prefix_len [n_groups], the tokens they share, read through the table of the group's
    first sequence. max_query, max_group (new tokens of one sequence and of one group), max_prefix and max_own
    (tokens of a prefix and behind it) shape the launch; a step beyond them is computed too, only slower.
    """
    dev, batch = _ragged_batch(q, k_pool, v_pool, out, query_start, positions, block_tables, max_query, scale, workspace)
    for t in (group_start, prefix_len):
        if t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous():
            _refuse(dict(group_start=group_start, prefix_len=prefix_len), dev, torch.int32)
    n_groups = prefix_len.numel()
    if group_start.numel() != n_groups + 1:
        raise EmberError("group_start must be [n_groups + 1], for as many groups as prefix_len has")
    a = _lib.PrefixAttnArgs(*batch, group_start.data_ptr(), prefix_len.data_ptr(),
                            *_prefix_sizes(batch[8], n_groups, max_group, max_prefix, max_own, batch[10]))
    _launch(_lib.lib().ember_hip_shared_prefix_attn, a, dev, stream, "shared_prefix_attn")
    return out


def kv4_pool(num_blocks: int, n_kv: int, device="cuda"):
    """A layer's pool of 4-bit pages, zeros: uint8 [num_blocks, n_kv, KV4_PAGE_BYTES], K and V together. Whole pages are
    copied by indexing (pool[dst] = pool[src])."""
    return torch.zeros(num_blocks, n_kv, KV4_PAGE_BYTES, dtype=torch.uint8, device=device)


def kv4_append(qkv, q_out, pool, positions, token_seq, block_tables, *, n_heads, n_kv, inv_freq_dev, q_norm=None,
               k_norm=None, bias=None, eps=1e-6, k_out=None, v_out=None, stream=None):
    """QK-RMSNorm + RoPE + the write of K and V into 4-bit pages, for one layer (ember_hip_kv4_append).

    qkv f16 [T, (n_heads + 2 n_kv) * 128] and q_out f16 [T, n_heads * 128] (any shape of that size); pool of kv4_pool;
    positions [T], token_seq [T] (rows of block_tables) and block_tables [rows, max_blocks] int32 on the device, as
    step_tables writes them. q_norm, k_norm [128], bias and inv_freq_dev [64] f32. k_out, v_out: None, or f16
    [T, n_kv * 128], which get what the codes stand for.
    """
    dev, f16, f32, i32 = qkv.get_device(), torch.float16, torch.float32, torch.int32
    if dev < 0:
        raise EmberError(f"qkv must be a device tensor (got {qkv.device})")
    _check_kv4_pool(pool, dev)
    for t in (qkv, q_out):
        if t.dtype is not f16 or t.get_device() != dev or not t.is_contiguous():
            _refuse(dict(qkv=qkv, q_out=q_out), dev, f16)
    for t in (positions, token_seq, block_tables):
        if t.dtype is not i32 or t.get_device() != dev or not t.is_contiguous():
            _refuse(dict(positions=positions, token_seq=token_seq, block_tables=block_tables), dev, i32)
    T, width, table, blocks = positions.numel(), (n_heads + 2 * n_kv) * HEAD_DIM, block_tables.shape, pool.shape
    if qkv.numel() != T * width or q_out.numel() != T * n_heads * HEAD_DIM or token_seq.numel() != T:
        raise EmberError("qkv, q_out and token_seq must hold as many tokens as positions")
    if blocks[1] != n_kv or len(table) != 2:
        raise EmberError("pool must have n_kv heads and block_tables be [rows, max_blocks]")
    floats = (inv_freq_dev,) if q_norm is None and k_norm is None and bias is None else (inv_freq_dev, q_norm, k_norm, bias)
    at = [0, 0, 0, 0]
    for i, t in enumerate(floats):
        if t is not None:
            if t.dtype is not f32 or t.get_device() != dev or not t.is_contiguous():
                _refuse({("inv_freq_dev", "q_norm", "k_norm", "bias")[i]: t}, dev, f32)
            if t.numel() != (HEAD_DIM // 2, HEAD_DIM, HEAD_DIM, width)[i]:
                raise EmberError(f"{('inv_freq_dev', 'q_norm', 'k_norm', 'bias')[i]} must hold {(HEAD_DIM // 2, HEAD_DIM, HEAD_DIM, width)[i]} values")
            at[i] = t.data_ptr()
    k_at = v_at = 0
    if k_out is not None or v_out is not None:
        for name, t in (("k_out", k_out), ("v_out", v_out)):
            if t is None:
                raise EmberError("k_out and v_out go together")
            if t.dtype is not f16 or t.get_device() != dev or not t.is_contiguous():
                _refuse({name: t}, dev, f16)
            if t.numel() != T * n_kv * HEAD_DIM:
                raise EmberError(f"{name} must hold {T * n_kv * HEAD_DIM} values")
        k_at, v_at = k_out.data_ptr(), v_out.data_ptr()
    a = _lib.Kv4AppendArgs(qkv.data_ptr(), q_out.data_ptr(), pool.data_ptr(), k_at, v_at, at[1], at[2], at[3], at[0],
                           positions.data_ptr(), token_seq.data_ptr(), block_tables.data_ptr(), table[0], table[1], T, n_heads, n_kv,
                           HEAD_DIM, blocks[0], eps)
    _launch(_lib.lib().ember_hip_kv4_append, a, dev, stream, "kv4_append")


def kv4_workspace(T: int, S: int, *, n_heads, n_kv, max_query=None, max_context=None, max_blocks=None, device="cuda",
                  stream=None):
    """A workspace (zeros) for kv4_attention of batches of these sizes and smaller ones, or None when no such call splits
    its keys. Only kv4_attention may write to it: not a workspace of the other attentions, which keep nothing between
    calls. It is zeroed in the order of `stream` (None: torch's current one); calls on another stream wait for that."""
    a = _lib.Kv4AttnArgs(*_batch_sizes(T, S, n_heads, n_kv, max_query, torch.float16, max_blocks),
                         _context(max_context, 1 << 26 if max_blocks is None else max_blocks))
    n = _workspace_bytes(_lib.lib().ember_hip_kv4_workspace_bytes, a)
    return _new_on(device, stream, torch.zeros, n) if n > 0 else None


def _context(max_context, max_blocks):
    if max_context is None:
        return max(1, min(max_blocks * BLOCK_SIZE, 0x7FFFFFFF))
    if not 0 < max_context <= 0x7FFFFFFF:
        raise EmberError(f"max_context must be 1 .. 2^31 - 1 (got {max_context})")
    return max_context


def kv4_attention(q, pool, out, query_start, positions, block_tables, *, max_query=None, max_context=None, scale=None,
                  workspace=None, stream=None):
    """Causal attention of a ragged batch over 4-bit pages (ember_hip_kv4_attn); returns out.

    q f16 [T, n_heads, 128] (a part of wider rows is fine), out the same, contiguous; pool of kv4_pool; query_start
    [S + 1], positions [T] and block_tables [S, max_blocks] int32 on the device, as step_tables writes them. Rows of
    q past query_start[S] are left alone. max_query and max_context: the most tokens and keys of one sequence (None:
    T, the tables' width); a step beyond them is computed too, only slower. workspace: of kv4_workspace, not shared
    by calls that overlap in time (None: no splits).
    """
    if q.dtype is not torch.float16:
        raise EmberError(f"q must be f16 (got {q.dtype})")
    dev, batch = _ragged_batch(q, pool, None, out, query_start, positions, block_tables, max_query, scale, workspace)
    _launch(_lib.lib().ember_hip_kv4_attn, _lib.Kv4AttnArgs(*batch, _context(max_context, batch[10])), dev, stream, "kv4_attn")
    return out


def mx_quantize(x, stream=None):
    """Rows to 4 bits (ember_hip_mx_quantize): f16 or f32 [rows, cols], cols a multiple of 32, rows of any stride from cols.
    Returns codes uint8 [rows, cols / 2] (byte i: columns 2i, in the low four bits, and 2i + 1) and scales uint8
    [rows, cols / 32]: value = (0, 0.5, 1, 1.5, 2, 3, 4, 6)[code % 8] * (-1 if code > 7) * 2^(scale - 127)."""
    dev = x.get_device()
    if dev < 0 or x.dim() != 2 or not (x.dtype is torch.float16 or x.dtype is torch.float32) or (x.shape[1] > 1 and x.stride(1) != 1):
        raise EmberError("mx_quantize: x must be an f16 or f32 device tensor [rows, cols] with contiguous rows")
    rows, cols = x.shape
    codes, scales = (_new_on(x.device, stream, torch.empty, rows, n) for n in (cols // 2, cols // _lib.MX_GROUP))
    a = _lib.MxQuantizeArgs(x.data_ptr(), x.stride(0) if rows > 1 else cols, rows, cols, _dtype_code(x), codes.data_ptr(),
                            scales.data_ptr())
    _launch(_lib.lib().ember_hip_mx_quantize, a, dev, stream, "mx_quantize")
    return codes, scales


def gemv4_pack(codes, scales, stream=None):
    """A 4-bit weight [N, K] as mx_quantize returns it (or a checkpoint in that format) laid out for gemv4: a flat uint8
    device tensor."""
    dev = codes.get_device()
    if dev < 0 or codes.dim() != 2 or scales.dim() != 2:
        raise EmberError("gemv4_pack: codes [N, K / 2] and scales [N, K / 32] must be device tensors")
    _refuse(dict(codes=codes, scales=scales), dev, torch.uint8)
    N, K = codes.shape[0], codes.shape[1] * 2
    if scales.shape != (N, K // _lib.MX_GROUP):
        raise EmberError(f"gemv4_pack: scales must be [{N}, {K // _lib.MX_GROUP}]")
    n = int(_lib.lib().ember_hip_gemv4_packed_bytes(N, K))
    if n <= 0:
        raise EmberError(_lib.last_error())
    out = _new_on(codes.device, stream, torch.empty, n)
    fn = _lib.lib().ember_hip_gemv4_pack
    _launch(lambda args, handle: fn(*args, handle), (codes.data_ptr(), scales.data_ptr(), N, K, out.data_ptr()), dev, stream, "gemv4_pack")
    return out


def gemv4(a, packed, c, epilogue: int, *, N: int, stream=None):
    """C = epilogue(A . W^T) with W [N, K] of gemv4_pack (ember_hip_gemv4).

    a: f16 [M, K] (rows of any stride from K that is a multiple of 8), up to 2^21 rows; c: as gemv's, rows of any stride
    from its width, apart from a. packed is known by its size alone: N and K are the caller's to get right. A row's bits
    do not depend on the other rows.
    """
    dev, shape, stride = a.get_device(), a.shape, a.stride()
    if dev < 0 or a.dtype is not torch.float16 or len(shape) != 2 or stride[1] != 1:
        raise EmberError("gemv4: a must be an f16 device tensor [M, K] with contiguous rows")
    M, K = shape
    if packed.dtype is not torch.uint8 or packed.get_device() != dev or not packed.is_contiguous():
        _refuse(dict(packed=packed), dev, torch.uint8)
    if packed.nbytes != (N + 15) // 16 * ((K + 127) // 128) * 1088 or packed.nbytes == 0:  # as ember_hip_gemv4_packed_bytes
        raise EmberError(f"gemv4: packed is not a weight of [{N}, {K}]")
    cols = N // 2 if epilogue == _lib.EPILOGUE_SILU_MUL else N
    want = torch.float32 if epilogue == _lib.EPILOGUE_STORE_F32 or epilogue == _lib.EPILOGUE_ADD_F32 else torch.float16
    rows = c.stride()
    if c.dtype is not want or c.get_device() != dev or c.shape != (M, cols) or (cols > 1 and rows[1] != 1):
        raise EmberError(f"gemv4: c must be {want} [{M}, {cols}] on cuda:{dev} with contiguous rows")
    _launch(_lib.lib().ember_hip_gemv4, _lib.Gemv4Args(a.data_ptr(), stride[0] if M > 1 else K, packed.data_ptr(), M, N, K, c.data_ptr(),
                                                       rows[0] if M > 1 else cols, epilogue), dev, stream, "gemv4")
