// Attention of ragged batches over spans of the paged cache: a window and the
// first tokens (ember_hip_window_attn), or a prefix that a group of sequences
// shares and each sequence's own keys behind it (ember_hip_shared_prefix_attn).
//
// A query row (token, head of the kv head's G) at position p sees key j iff
//   base <= j <= min(p, limit - 1)  and  (p - j < window  or  j < sinks);
// a launch is phases of that one rule:
//   window   rows of one sequence, base 0, no limit;
//   prefix   rows of all sequences of a group, limit = the prefix's length,
//            through the first sequence's table;
//   own      rows of one sequence, base = its group's prefix length.
// The pages that hold such keys are at most two runs of the table (the first
// tokens' and the rest), numbered through as virtual pages, so no other entry
// of the table is followed and a split is a run of virtual pages. Rows that
// are split (over a long axis, or into prefix and own keys) leave partials
// (running max, sum, unnormalised output) in slots of the workspace, which a
// merge launch joins in slot order: no atomics, the same bits every time.
//
// Two forms. Few rows (16 at most: decode, verify) are bound by the read of
// the pages: span_walk_kernel gives each wave pages of its own, straight from
// HBM. Many rows (prompt chunks, a group's rows before a long prefix) are bound by
// the products: span_tile_kernel shares 64-key blocks in LDS between waves of
// 32 rows each.
#include <algorithm>
#include <climits>

#include "capi_errors.hpp"
#include "device.hpp"
#include "kernels.hpp"
#include "paged_device.hpp"

namespace ember::hip {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kWalkRows = 16;              // query rows of a walk work-group: one MFMA column each
constexpr int kTileRows = 32 * kWaves;     // query rows of a tile work-group: 32 a wave
constexpr int kBlockPages = 4;             // pages of a tile's key block
constexpr int kBlockKeys = kBlockPages * kPage;
constexpr int kNoWindow = INT_MAX;

enum Kind : int { kWindowRows, kPrefixRows, kOwnRows };

// One phase of a launch: `units` sequences (or groups), each `tiles` row tiles (a work-group takes every tiles-th
// from its own on), each `splits` runs of `pages` virtual pages (the last run takes what is left). Its partials go
// to slots slot0 .. slot0 + splits - 1.
struct Phase {
    int kind, units, tiles, splits, pages, slot0;
};

struct SpanParams {
    const void *q, *k, *v;
    void *out;
    const int32_t *query_start, *positions, *tables, *group_start, *prefix_len;
    float *part_acc, *part_ml;  // [T, n_heads, slots][128], [T, n_heads, slots][2]
    int64_t q_stride;
    int T, S, max_blocks, n_heads, n_kv, G, num_blocks, n_groups, window, sinks, slots;
    float scale_log2;
};

__device__ __forceinline__ int clamped(int x, int most) { return min(max(x, 0), most); }

// The rows of one work item and the bounds of the keys they see.
struct Rows {
    int t0, rows;     // first token, (token, head) rows
    int seq;          // the table's row
    int base, limit;  // keys base .. limit - 1
};

// The prefix length of sequence s's group; 0 if it is in none. 64 starts are looked at together, so up to 4096
// groups cost two loads one after the other.
__device__ __forceinline__ int own_base(const SpanParams &p, int s, int lane, bool &grouped) {
    int lo = 0, n = p.n_groups;  // the group, if there is one, is among lo .. lo + n - 1
    while (n > 0) {
        const int step = (n + kWave - 1) / kWave;
        const int at = lo + lane * step;
        const bool starts = lane * step < n && p.group_start[at] <= s;
        const int c = __popcll(__builtin_amdgcn_ballot_w64(starts));  // starts are ascending: lanes 0 .. c - 1
        if (c == 0) break;
        const int from = uniform(lo + (c - 1) * step);
        if (step == 1) {
            grouped = s < uniform_load(p.group_start + from + 1);
            return grouped ? max(0, uniform_load(p.prefix_len + from)) : 0;
        }
        n = min(step, lo + n - from);
        lo = from;
    }
    grouped = false;
    return 0;
}

__device__ __forceinline__ Rows rows_of(const SpanParams &p, const Phase &ph, int unit, int lane, bool &grouped) {
    Rows r;
    int s0 = unit, s1 = unit + 1;
    r.base = 0;
    r.limit = INT_MAX;
    grouped = true;
    if (ph.kind == kPrefixRows) {
        s0 = clamped(uniform_load(p.group_start + unit), p.S);
        s1 = clamped(uniform_load(p.group_start + unit + 1), p.S);
        r.limit = max(0, uniform_load(p.prefix_len + unit));
    } else if (ph.kind == kOwnRows) {
        r.base = own_base(p, unit, lane, grouped);
    }
    r.t0 = clamped(uniform_load(p.query_start + s0), p.T);
    r.rows = max(0, clamped(uniform_load(p.query_start + s1), p.T) - r.t0) * p.G;
    r.seq = min(s0, p.S - 1);
    if (s1 <= s0) r.rows = 0;
    return r;
}

// The virtual pages of rows at positions min_pos .. max_pos whose highest visible keys are at most max_top.
struct Span {
    int lo;       // the first key that a window reaches
    int head;     // virtual pages 0 .. head - 1 are the table's first ones; page v >= head is the table's v + skip
    int skip, pages;
    __device__ __forceinline__ int page(int v) const { return v < head ? v : v + skip; }
};

__device__ __forceinline__ Span span_of(const Rows &r, int window, int sinks, int min_pos, int max_top) {
    Span s;
    s.lo = max(r.base, window == kNoWindow ? 0 : min_pos - window + 1);
    s.lo = max(s.lo, 0);
    const int first = s.lo / kPage;
    s.head = min((max(min(sinks, max_top + 1), 0) + kPage - 1) / kPage, first);
    s.skip = first - s.head;
    s.pages = s.head + (s.lo <= max_top ? max_top / kPage - first + 1 : 0);
    return s;
}

// Whether every key of a page is visible to every row (positions min_pos .. max_pos, highest keys at least min_top).
__device__ __forceinline__ bool whole_page(int page, const Rows &r, int window, int sinks, int max_pos, int min_top) {
    const int j0 = page * kPage;
    return j0 >= r.base && j0 + kPage - 1 <= min_top && (max_pos - j0 < window || j0 + kPage <= sinks);
}

__device__ __forceinline__ bool visible(int j, int base, int top, int pos, int window, int sinks) {
    return j >= base && j <= top && (pos - j < window || j < sinks);
}

// ---- few rows: a page per wave ----

// Lane l = 16 g + c serves query column c, the item's row c (columns past the last repeat it). The f16 form is
// the decode kernel's: S^T = K Q^T on v_mfma_f32_16x16x32_f16 with the keys staged in the wave's LDS by direct
// loads, O^T += V^T P^T on v_mfma_f32_16x16x16_f16 with V in registers. f32 pages use v_mfma_f32_16x16x4_f32 the
// same way: step s of the scores takes dim 16 (s / 4) + 4 g + s % 4 from lane group g, so a lane loads key c in
// 16-byte pieces; step v of the values takes key 4 g + v, which the lane's own scores belong to.
template <typename T>
struct WalkPage;
template <>
struct WalkPage<f16> {
    u32x4 v[4];  // keys 4 g + i, dims 8 c .. 8 c + 7
};
template <>
struct WalkPage<float> {
    u32x4 k[8];     // key c, dims 16 i + 4 g .. + 3
    u32x4 v[4][2];  // keys 4 g + i, dims 8 c .. 8 c + 7
};

template <typename T>
__device__ __forceinline__ void walk_item(const SpanParams &p, const Phase &ph, const int id) {
    constexpr int D = kHeadDim;
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int RP = D + 4;            // floats of a row's partial in LDS: 16 rows' pieces of one dim on distinct banks
    constexpr int RW = kWalkRows * RP;   // floats of a wave's region (its first 4 KiB also stage f16 keys)
    __shared__ __align__(16) float red[kWaves * RW];
    __shared__ float red_m[kWalkRows][kWaves], red_l[kWalkRows][kWaves];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int g = lane >> 4, c = lane & 15;
    const int kvh = id % p.n_kv;
    int rest = id / p.n_kv;
    const int split = rest % ph.splits;
    rest /= ph.splits;
    const int tile0 = rest % ph.tiles, unit = rest / ph.tiles;

    bool grouped;
    const Rows r = rows_of(p, ph, unit, lane, grouped);
    const int32_t *const table = p.tables + static_cast<int64_t>(r.seq) * p.max_blocks;
    const int64_t head_off = static_cast<int64_t>(kvh) * (kPage * D), block_stride = static_cast<int64_t>(p.n_kv) * (kPage * D);
    const T *const kbase = static_cast<const T *>(p.k) + head_off, *const vbase = static_cast<const T *>(p.v) + head_off;
    const int window = ph.kind == kWindowRows ? p.window : kNoWindow, sinks = ph.kind == kWindowRows ? p.sinks : 0;

    for (int row0 = tile0 * kWalkRows; row0 < r.rows; row0 += ph.tiles * kWalkRows) {
        const int nrows = min(kWalkRows, r.rows - row0);
        const int my_row = row0 + min(c, nrows - 1);
        const int my_tok = r.t0 + my_row / p.G, my_head = kvh * p.G + my_row % p.G;
        const int my_pos = max(p.positions[my_tok], -1);
        // The row's q as the scores' B operand; used after the first pages are on their way.
        u32x4 qf[F16 ? 4 : 8];
        {
            const T *qp = static_cast<const T *>(p.q) + my_tok * p.q_stride + my_head * D;
#pragma unroll
            for (int i = 0; i < (F16 ? 4 : 8); i++)
                qf[i] = *reinterpret_cast<const u32x4 *>(qp + (F16 ? 32 * i + 8 * g : 16 * i + 4 * g));
        }
        const int my_top = min(min(my_pos, r.limit - 1), p.max_blocks * kPage - 1);
        int min_pos = my_pos, max_pos = my_pos, min_top = my_top, max_top = my_top;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            min_pos = min(min_pos, __shfl_xor(min_pos, o, kWave));
            max_pos = max(max_pos, __shfl_xor(max_pos, o, kWave));
            min_top = min(min_top, __shfl_xor(min_top, o, kWave));
            max_top = max(max_top, __shfl_xor(max_top, o, kWave));
        }
        min_pos = uniform(min_pos), max_pos = uniform(max_pos), min_top = uniform(min_top), max_top = uniform(max_top);
        const Span sp = span_of(r, window, sinks, min_pos, max_top);
        const int v0 = min(split * ph.pages, sp.pages);
        const int v1 = split == ph.splits - 1 ? sp.pages : min(v0 + ph.pages, sp.pages);

        float mc = kNoMax, lc = 0.0f;
        f32x4 o[8];  // o[t][v]: dim 32 g + 8 v + t of column c
#pragma unroll
        for (int t = 0; t < 8; t++) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t *const kstage = reinterpret_cast<uint32_t *>(&red[wave * RW]);
        uint32_t k_dma[4], k_rd[4];  // f16: the swizzled stage (slot 16 k + (q ^ k): chunk q of key k), bytes and dwords
#pragma unroll
        for (int i = 0; i < 4; i++) {
            k_dma[i] = 1024u * i + 256u * g + 16u * ((c ^ (4 * i + g)) & 15);
            k_rd[i] = 64u * c + 4u * (((4 * i + g) ^ c) & 15);
        }
        // The block ids of up to 64 virtual pages, one a lane; wave w takes pages w, w + 4, ...
        for (int cv = v0; cv < v1; cv += kWave) {
            const int chunk = min(kWave, v1 - cv);
            const int n = chunk > wave ? (chunk - 1 - wave) / kWaves + 1 : 0;
            const int ids = lane < chunk ? table[sp.page(cv + lane)] : -1;
            auto desc_of = [&](const T *base, int j) {
                const int blk = __builtin_amdgcn_readlane(ids, min(wave + j * kWaves, chunk - 1));
                const bool live = j < n && blk >= 0 && blk < p.num_blocks;  // dead: no records, the loads give zeros
                return __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base) + (live ? blk : 0) * block_stride, 0,
                                                         live ? kPage * D * static_cast<int>(sizeof(T)) : 0, kDescWord3);
            };
            WalkPage<T> A;
            auto fetch_keys = [&](int j) {
                const __amdgpu_buffer_rsrc_t d = desc_of(kbase, j);
                if constexpr (F16) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(
                            d, (__attribute__((address_space(3))) void *)(kstage + 256 * i), 16, k_dma[i], 0, 0, kNonTemporal);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) A.k[i] = load_desc(d, 512u * c + 64u * i + 16u * g);
                }
            };
            auto fetch_values = [&](int j) {
                const __amdgpu_buffer_rsrc_t d = desc_of(vbase, j);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (F16) {
                        A.v[i] = load_desc(d, 1024u * g + 256u * i + 16u * c);
                    } else {
                        A.v[i][0] = load_desc(d, 2048u * g + 512u * i + 32u * c);
                        A.v[i][1] = load_desc(d, 2048u * g + 512u * i + 32u * c + 16u);
                    }
                }
            };
            fetch_keys(0);
            fetch_values(0);
            for (int j = 0; j < n; j++) {
                const int page = sp.page(cv + wave + j * kWaves);
                f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};  // s[v]: raw score of key 4 g + v
                if constexpr (F16) {
                    u32x4 kf[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) kf[i] = *reinterpret_cast<const u32x4 *>(kstage + k_rd[i]);
#pragma unroll
                    for (int i = 0; i < 4; i++) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(kf[i]), as_f16x8(qf[i]), s, 0, 0, 0);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(A.k[i][e]), __uint_as_float(qf[i][e]), s, 0, 0, 0);
                }
                uint32_t dead = 0;  // bit v: no row sees key 4 g + v, whose values may then be anything
                if (!whole_page(page, r, window, sinks, max_pos, min_top)) {
                    const int key0 = page * kPage + 4 * g;
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const bool see = visible(key0 + v, r.base, my_top, my_pos, window, sinks);
                        s[v] = see ? s[v] : -INFINITY;
                        const uint64_t rows_that_see = __builtin_amdgcn_ballot_w64(see);
                        dead |= (rows_that_see >> (16 * g) & 0xffff) == 0 ? 1u << v : 0u;
                    }
                }
                // Online softmax in base 2, the scale in the exponent. mc starts finite, so a row that has seen
                // nothing yet keeps weight sums of 0 and corrections of 1.
                const float mn = fmaxf(mc, groups_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))) * p.scale_log2);
                const float corr = exp2_hw(mc - mn);
                mc = mn;
                float w[4];
#pragma unroll
                for (int v = 0; v < 4; v++) w[v] = exp2_hw(__builtin_fmaf(s[v], p.scale_log2, -mn));
                // f16: the weights are rounded to f16, the products' operand, and summed as rounded, so that the
                // rounding of a weight (2^-12 of it at most) moves numerator and denominator alike.
                f16x4 wh;
                if constexpr (F16) {
#pragma unroll
                    for (int v = 0; v < 4; v++) wh[v] = static_cast<f16>(w[v]);
                    const f16x2 ones = {static_cast<f16>(1.0f), static_cast<f16>(1.0f)};
                    lc = __builtin_amdgcn_fdot2(wh.zw, ones, __builtin_amdgcn_fdot2(wh.xy, ones, lc * corr, false), false);
                } else {
                    lc = lc * corr + ((w[0] + w[1]) + (w[2] + w[3]));
                }
#pragma unroll
                for (int t = 0; t < 8; t++) o[t] = o[t] * corr;
                __builtin_amdgcn_sched_barrier(0);
                fetch_keys(j + 1);
                __builtin_amdgcn_sched_barrier(0);
                if (__builtin_amdgcn_ballot_w64(dead != 0)) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool drop = dead >> i & 1;
                        if constexpr (F16) {
                            A.v[i] = drop ? u32x4{0, 0, 0, 0} : A.v[i];
                        } else {
                            A.v[i][0] = drop ? u32x4{0, 0, 0, 0} : A.v[i][0];
                            A.v[i][1] = drop ? u32x4{0, 0, 0, 0} : A.v[i][1];
                        }
                    }
                }
                if constexpr (F16) {
                    o[0] = __builtin_amdgcn_mfma_f32_16x16x16f16(value_tile<0>(A.v), wh, o[0], 0, 0, 0);
                    o[1] = __builtin_amdgcn_mfma_f32_16x16x16f16(value_tile<1>(A.v), wh, o[1], 0, 0, 0);
                    o[2] = __builtin_amdgcn_mfma_f32_16x16x16f16(value_tile<2>(A.v), wh, o[2], 0, 0, 0);
                    o[3] = __builtin_amdgcn_mfma_f32_16x16x16f16(value_tile<3>(A.v), wh, o[3], 0, 0, 0);
                    o[4] = __builtin_amdgcn_mfma_f32_16x16x16f16(value_tile<4>(A.v), wh, o[4], 0, 0, 0);
                    o[5] = __builtin_amdgcn_mfma_f32_16x16x16f16(value_tile<5>(A.v), wh, o[5], 0, 0, 0);
                    o[6] = __builtin_amdgcn_mfma_f32_16x16x16f16(value_tile<6>(A.v), wh, o[6], 0, 0, 0);
                    o[7] = __builtin_amdgcn_mfma_f32_16x16x16f16(value_tile<7>(A.v), wh, o[7], 0, 0, 0);
                } else {
#pragma unroll
                    for (int v = 0; v < 4; v++)
#pragma unroll
                        for (int t = 0; t < 8; t++)
                            o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(A.v[v][t / 4][t % 4]), w[v], o[t], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                fetch_values(j + 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            // The fetch past the last page still writes zeros into the stage, where the next chunk's keys or the
            // wave's partial go.
            __builtin_amdgcn_s_waitcnt(0);
        }

        // The column's sum over its lane groups, the wave's partial into LDS, and the waves' merge in order.
        lc = groups_sum(lc);
        if (c < nrows) {
#pragma unroll
            for (int v = 0; v < 4; v++) {
                float *dst = &red[wave * RW + c * RP + 32 * g + 8 * v];
                *reinterpret_cast<float4 *>(dst) = make_float4(o[0][v], o[1][v], o[2][v], o[3][v]);
                *reinterpret_cast<float4 *>(dst + 4) = make_float4(o[4][v], o[5][v], o[6][v], o[7][v]);
            }
            if (g == 0) {
                red_m[c][wave] = mc;
                red_l[c][wave] = lc;
            }
        }
        __syncthreads();
        for (int idx = tid; idx < nrows * D; idx += kThreads) {
            const int row = idx / D, d = idx % D;
            float M = kNoMax;
#pragma unroll
            for (int w = 0; w < kWaves; w++) M = fmaxf(M, red_m[row][w]);
            float L = 0.0f, O = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                const float f = exp2_hw(red_m[row][w] - M);
                L = L + red_l[row][w] * f;
                O = O + red[w * RW + row * RP + d] * f;
            }
            const int tok = r.t0 + (row0 + row) / p.G, head = kvh * p.G + (row0 + row) % p.G;
            const int64_t at = static_cast<int64_t>(tok) * p.n_heads + head;
            if (p.slots == 1) {
                static_cast<T *>(p.out)[at * D + d] = from_f32<T>(L > 0.0f ? O / L : 0.0f);
            } else {
                const int64_t slot = at * p.slots + ph.slot0 + split;
                p.part_acc[slot * D + d] = O;
                if (d == 0) {
                    p.part_ml[slot * 2] = M;
                    p.part_ml[slot * 2 + 1] = L;
                    // rows of no group: their prefix slots hold nothing
                    if (!grouped && split == 0)
                        for (int i = 0; i < ph.slot0; i++) {
                            p.part_ml[(at * p.slots + i) * 2] = kNoMax;
                            p.part_ml[(at * p.slots + i) * 2 + 1] = 0.0f;
                        }
                }
            }
        }
        __syncthreads();  // the regions are the next row tile's stages
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) span_walk_kernel(SpanParams p, Phase a, Phase b, int a_groups) {
    const int id = static_cast<int>(blockIdx.x);
    const bool second = id >= a_groups;
    walk_item<T>(p, second ? b : a, second ? id - a_groups : id);
}

// ---- many rows: key blocks shared in LDS (f16) ----

// Wave w owns rows 32 w .. 32 w + 31 of the tile; lane l = 32 h + c serves row c.
//   S^T = K Q^T   v_mfma_f32_32x32x16_f16: lane l ends with row c's scores of keys 8 (i / 4) + 4 h + i % 4 of each
//                 32-key half, i = 0 .. 15, so a row lives in two lanes: its max and sum meet through one
//                 v_permlane32_swap, and rescaling O touches no other lane.
//   O^T += V^T P^T  the lane's scores, as weights in f16, are the B operand as they stand (the order of the keys
//                 inside one product is free); the A operand, the same keys of dim c, comes from the transposing
//                 LDS read: lane r of a 16-lane block reads four dims of key r / 4, lane i receives dim i of 4 keys.
constexpr int kRow = kHeadDim + 16;  // LDS row of a key, halves: 72 dwords, so 8 rows start 8 banks apart
typedef __fp16 tr16x4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __attribute__((address_space(3))) tr16x4 lds_tr16x4;

// How far (base 2) a score may pass the reference max before the reference moves: weights stay below 2^8, which
// f16 holds, and most blocks rescale nothing.
constexpr float kLazy = 8.0f;

__global__ void __launch_bounds__(kThreads, 2) span_tile_kernel(SpanParams p, Phase ph) {
    constexpr int D = kHeadDim;
    __shared__ __align__(16) f16 k_lds[2][kBlockKeys * kRow], v_lds[2][kBlockKeys * kRow];
    __shared__ int ext[kWaves][4];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int h = lane >> 5, c = lane & 31;
    const int id = static_cast<int>(blockIdx.x);
    const int kvh = id % p.n_kv;
    int rest = id / p.n_kv;
    const int split = rest % ph.splits;
    rest /= ph.splits;
    const int tile0 = rest % ph.tiles, unit = rest / ph.tiles;

    bool grouped;
    const Rows r = rows_of(p, ph, unit, lane, grouped);
    const int32_t *const table = p.tables + static_cast<int64_t>(r.seq) * p.max_blocks;
    const int64_t head_off = static_cast<int64_t>(kvh) * (kPage * D), block_stride = static_cast<int64_t>(p.n_kv) * (kPage * D);
    const f16 *const kbase = static_cast<const f16 *>(p.k) + head_off, *const vbase = static_cast<const f16 *>(p.v) + head_off;
    const int window = ph.kind == kWindowRows ? p.window : kNoWindow, sinks = ph.kind == kWindowRows ? p.sinks : 0;

    for (int row0 = tile0 * kTileRows; row0 < r.rows; row0 += ph.tiles * kTileRows) {
        const int my_row = min(row0 + 32 * wave + c, r.rows - 1);  // rows past the last repeat it
        const bool mine = row0 + 32 * wave + c < r.rows;
        const int my_tok = r.t0 + my_row / p.G, my_head = kvh * p.G + my_row % p.G;
        const int my_pos = max(p.positions[my_tok], -1);
        f16x8 qf[8];
        {
            const f16 *qp = static_cast<const f16 *>(p.q) + my_tok * p.q_stride + my_head * D;
#pragma unroll
            for (int i = 0; i < 8; i++) qf[i] = *reinterpret_cast<const f16x8 *>(qp + 16 * i + 8 * h);
        }
        const int my_top = min(min(my_pos, r.limit - 1), p.max_blocks * kPage - 1);
        int lo_pos = my_pos, hi_pos = my_pos, lo_top = my_top, hi_top = my_top;  // of the wave
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            lo_pos = min(lo_pos, __shfl_xor(lo_pos, o, kWave));
            hi_pos = max(hi_pos, __shfl_xor(hi_pos, o, kWave));
            lo_top = min(lo_top, __shfl_xor(lo_top, o, kWave));
            hi_top = max(hi_top, __shfl_xor(hi_top, o, kWave));
        }
        lo_pos = uniform(lo_pos), hi_pos = uniform(hi_pos), lo_top = uniform(lo_top), hi_top = uniform(hi_top);
        if (lane == 0) ext[wave][0] = lo_pos, ext[wave][1] = hi_top;
        __syncthreads();
        int min_pos = lo_pos, max_top = hi_top;  // of the tile
#pragma unroll
        for (int w = 0; w < kWaves; w++) min_pos = min(min_pos, ext[w][0]), max_top = max(max_top, ext[w][1]);
        min_pos = uniform(min_pos), max_top = uniform(max_top);
        const Span sp = span_of(r, window, sinks, min_pos, max_top);
        const int v0 = min(split * ph.pages, sp.pages);
        const int v1 = split == ph.splits - 1 ? sp.pages : min(v0 + ph.pages, sp.pages);
        const int blocks = (v1 - v0 + kBlockPages - 1) / kBlockPages;

        float m = -INFINITY, l = 0.0f;
        f32x16 o[4];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] = 0.0f;

        // A block's pages into registers: each page one 16-byte piece a thread, of key tid / 16. Keys that no row of
        // the tile sees may hold anything: their values become zeros, so that a zero weight meets no NaN.
        u32x4 kr[kBlockPages], vr[kBlockPages];
        int ids = -1, next_ids = v0 + lane < v1 ? table[sp.page(v0 + lane)] : -1;  // 64 virtual pages, one a lane
        auto fetch = [&](int b) {
            if (b % (kWave / kBlockPages) == 0) {
                ids = next_ids;
                const int v = v0 + b * kBlockPages + kWave + lane;
                next_ids = v < v1 ? table[sp.page(v)] : -1;
            }
#pragma unroll
            for (int j = 0; j < kBlockPages; j++) {
                const int v = v0 + b * kBlockPages + j;
                const int blk = __builtin_amdgcn_readlane(ids, (b * kBlockPages + j) % kWave);
                const bool live = v < v1 && blk >= 0 && blk < p.num_blocks;
                const int64_t at = (live ? blk : 0) * block_stride;
                const int bytes = live ? kPage * D * 2 : 0;
                const __amdgpu_buffer_rsrc_t kd = __builtin_amdgcn_make_buffer_rsrc(const_cast<f16 *>(kbase) + at, 0, bytes, kDescWord3);
                const __amdgpu_buffer_rsrc_t vd = __builtin_amdgcn_make_buffer_rsrc(const_cast<f16 *>(vbase) + at, 0, bytes, kDescWord3);
                kr[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kd, 16 * tid, 0, 0));
                vr[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vd, 16 * tid, 0, 0));
            }
        };
        auto stage = [&](int b) {
#pragma unroll
            for (int j = 0; j < kBlockPages; j++) {
                const int key = sp.page(v0 + b * kBlockPages + j) * kPage + tid / 16;
                const bool dead = key < r.base || key > max_top || (key < sp.lo && key >= sinks);
                const int at = (j * kPage + tid / 16) * kRow + tid % 16 * 8;
                *reinterpret_cast<u32x4 *>(&k_lds[b & 1][at]) = kr[j];
                *reinterpret_cast<u32x4 *>(&v_lds[b & 1][at]) = dead ? u32x4{0, 0, 0, 0} : vr[j];
            }
        };
        if (blocks > 0) {
            fetch(0);
            stage(0);
        }
        __syncthreads();
        for (int b = 0; b < blocks; b++) {
            if (b + 1 < blocks) fetch(b + 1);
            const f16 *const kl = k_lds[b & 1], *const vl = v_lds[b & 1];
            f32x16 s[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
#pragma unroll
                for (int i = 0; i < 16; i++) s[t][i] = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const f16x8 a = *reinterpret_cast<const f16x8 *>(&kl[(32 * t + c) * kRow + 16 * i + 8 * h]);
                    s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qf[i], s[t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int j = 0; j < kBlockPages; j++) {
                const int v = v0 + b * kBlockPages + j;
                const int page = sp.page(v);
                if (v < v1 && whole_page(page, r, window, sinks, hi_pos, lo_top)) continue;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = page * kPage + 8 * (i / 4) + 4 * h + i % 4;
                    const bool see = v < v1 && visible(key, r.base, my_top, my_pos, window, sinks);
                    s[j / 2][8 * (j % 2) + i] = see ? s[j / 2][8 * (j % 2) + i] : -INFINITY;
                }
            }
            float top = s[0][0];
#pragma unroll
            for (int i = 1; i < 32; i++) top = fmaxf(top, s[i / 16][i % 16]);
            top = top * p.scale_log2;
            if (__builtin_amdgcn_ballot_w64(top > m + kLazy)) {
                const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                const float row_top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
                const bool grow = row_top > m + kLazy;
                const float corr = grow ? exp2_hw(m - row_top) : 1.0f;  // 0 from a row that had seen nothing
                m = grow ? row_top : m;
                l = l * corr;
#pragma unroll
                for (int t = 0; t < 4; t++) o[t] = o[t] * corr;
            }
            const float neg = m == -INFINITY ? 0.0f : -m;
            f16x8 w[4];
            const f16x2 ones = {static_cast<f16>(1.0f), static_cast<f16>(1.0f)};
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    w[j][i] = static_cast<f16>(exp2_hw(__builtin_fmaf(s[j / 2][8 * (j % 2) + i], p.scale_log2, neg)));
#pragma unroll
                for (int i = 0; i < 4; i++) l = __builtin_amdgcn_fdot2(f16x2{w[j][2 * i], w[j][2 * i + 1]}, ones, l, false);
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const int r16 = lane & 15;
                    const f16 *const at = &vl[(16 * j + 4 * h + r16 / 4) * kRow + 32 * t + 16 * (lane >> 4 & 1) + 4 * (r16 % 4)];
                    const f16x4 lo4 = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr16x4 *)at));
                    const f16x4 hi4 = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr16x4 *)(at + 8 * kRow)));
                    const f16x8 a = {lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, w[j], o[t], 0, 0, 0);
                }
            if (b + 1 < blocks) stage(b + 1);
            __syncthreads();
        }

        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
        if (mine) {
            const int64_t at = static_cast<int64_t>(my_tok) * p.n_heads + my_head;
            if (p.slots == 1) {
                f16 *const dst = static_cast<f16 *>(p.out) + at * D + 4 * h;
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i++) {  // dims 32 (i / 4) + 8 (i % 4) + 4 h .. + 3
                    f16x4 x;
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = static_cast<f16>(o[i / 4][4 * (i % 4) + e] * inv);
                    *reinterpret_cast<f16x4 *>(dst + 8 * i) = x;
                }
            } else {
                const int64_t slot = at * p.slots + ph.slot0 + split;
                float *const dst = p.part_acc + slot * D + 4 * h;
#pragma unroll
                for (int i = 0; i < 16; i++)
                    *reinterpret_cast<float4 *>(dst + 8 * i) = make_float4(o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1],
                                                                           o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]);
                if (h == 0) {
                    p.part_ml[slot * 2] = l > 0.0f ? m : kNoMax;
                    p.part_ml[slot * 2 + 1] = l;
                }
            }
        }
    }
}

// ---- the slots' merge: a wave per (token, head), two dims a lane ----

template <typename T>
__global__ void __launch_bounds__(kThreads) span_merge_kernel(SpanParams p) {
    constexpr int D = kHeadDim;
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kWaves + uniform(static_cast<int>(threadIdx.x) / kWave);
    const int64_t tok = at / p.n_heads;
    if (tok < clamped(uniform_load(p.query_start), p.T) || tok >= clamped(uniform_load(p.query_start + p.S), p.T)) return;
    const float *const ml = p.part_ml + at * p.slots * 2;
    const float *const acc = p.part_acc + at * p.slots * D + 2 * lane;
    float M = kNoMax;
    for (int s = lane; s < p.slots; s += kWave) M = fmaxf(M, ml[2 * s]);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, kWave));
    float L = 0.0f, x = 0.0f, y = 0.0f;
    for (int s = 0; s < p.slots; s++) {
        const float ls = ml[2 * s + 1];
        if (!(ls > 0.0f)) continue;  // an empty slot's accumulators are not written
        const float f = exp2_hw(ml[2 * s] - M);
        const float2 a = *reinterpret_cast<const float2 *>(acc + static_cast<int64_t>(s) * D);
        L = L + ls * f;
        x = x + a.x * f;
        y = y + a.y * f;
    }
    T *const dst = static_cast<T *>(p.out) + at * D + 2 * lane;
    dst[0] = from_f32<T>(L > 0.0f ? x / L : 0.0f);
    dst[1] = from_f32<T>(L > 0.0f ? y / L : 0.0f);
}

// ---- host: phases and launches ----

// Cuts `pages` virtual pages into runs, for `items` work-groups per run: enough for `want` work-groups in all, each
// run at least `least` pages. Returns the runs that were allowed, which only grow with `pages` (the splits, equal
// runs of whole pages, need not): the workspace is sized by them.
int cut(Phase &ph, int64_t items, int pages, int want, int least) {
    const int64_t most = std::max(1, pages / least);
    const int64_t runs = std::clamp<int64_t>(want / std::max<int64_t>(1, items), 1, most);
    ph.pages = std::max<int>(1, static_cast<int>((pages + runs - 1) / runs));
    ph.splits = std::max(1, (pages + ph.pages - 1) / ph.pages);
    return static_cast<int>(runs);
}

struct Launch {
    Phase first{}, second{};  // second.units == 0: none
    bool first_tiled = false;
    int slots = 1, most_slots = 1;  // slots, and those that the workspace is sized for
};

int64_t groups_of(const Phase &ph, int n_kv) { return static_cast<int64_t>(ph.units) * ph.tiles * ph.splits * n_kv; }

int64_t partial_bytes(const EmberRaggedBatch &b, int slots) {
    return slots == 1 ? 0 : static_cast<int64_t>(b.T) * b.n_heads * slots * (kHeadDim + 2) * static_cast<int64_t>(sizeof(float));
}

int tiles_for(int64_t tokens, int G, int rows) { return static_cast<int>(std::max<int64_t>(1, (tokens * G + rows - 1) / rows)); }

// Work-groups wanted in a launch (two tile work-groups fill a CU's LDS and registers, four walk ones do) and the
// least pages worth a work-group of their own.
constexpr int kTileGroups = 512, kWalkGroups = 1024, kTileLeast = 16, kWalkLeast = 8;

// `spread` halves the work-groups asked for, step by step, until the workspace holds the partials.
Launch plan_window(const EmberWindowAttnArgs &a, int spread) {
    const EmberRaggedBatch &b = a.batch;
    const int G = b.n_heads / b.n_kv;
    const int64_t most = std::min(b.max_query, b.T);
    Launch l;
    l.first_tiled = b.dtype == EMBER_DTYPE_F16 && most * G > kWalkRows;
    const int rows = l.first_tiled ? kTileRows : kWalkRows;
    l.first = Phase{kWindowRows, b.S, tiles_for(most, G, rows), 1, 1, 0};
    // a tile's keys: the first tokens' pages, and the windows of its tokens
    const int64_t tokens = std::min<int64_t>(most, (rows + G - 1) / G + 1);
    const int64_t near = (std::min<int64_t>(a.window, static_cast<int64_t>(b.max_blocks) * kPage) + tokens + kPage - 1) / kPage + 1;
    const int pages = static_cast<int>(std::min<int64_t>(b.max_blocks, near + (static_cast<int64_t>(a.sinks) + kPage - 1) / kPage));
    l.most_slots = cut(l.first, static_cast<int64_t>(b.S) * l.first.tiles * b.n_kv, pages,
                       (l.first_tiled ? kTileGroups : kWalkGroups) >> spread, l.first_tiled ? kTileLeast : kWalkLeast);
    l.slots = l.first.splits;
    return l;
}

Launch plan_prefix(const EmberPrefixAttnArgs &a, int spread) {
    const EmberRaggedBatch &b = a.batch;
    const int G = b.n_heads / b.n_kv;
    const int64_t in_group = std::min(a.max_group, b.T), in_seq = std::min(b.max_query, b.T);
    auto pages_of = [&](int keys) { return std::min(b.max_blocks, keys / kPage + 2); };
    Launch l;
    l.first_tiled = b.dtype == EMBER_DTYPE_F16 && in_group * G > kWalkRows;
    if (a.n_groups > 0) {
        l.first = Phase{kPrefixRows, a.n_groups, tiles_for(in_group, G, l.first_tiled ? kTileRows : kWalkRows), 1, 1, 0};
        l.most_slots = cut(l.first, static_cast<int64_t>(a.n_groups) * l.first.tiles * b.n_kv, pages_of(a.max_prefix),
                           (l.first_tiled ? kTileGroups : kWalkGroups) >> spread, l.first_tiled ? kTileLeast : kWalkLeast);
    } else {
        l.most_slots = 0;
    }
    l.second = Phase{kOwnRows, b.S, tiles_for(in_seq, G, kWalkRows), 1, 1, l.first.splits};
    l.most_slots += cut(l.second, static_cast<int64_t>(b.S) * l.second.tiles * b.n_kv, pages_of(a.max_own),
                        kWalkGroups >> spread, kWalkLeast);
    l.slots = l.first.splits + l.second.splits;
    return l;
}
constexpr int kLeastSpread = 10;  // 1024 >> 10 = 1: no splits

SpanParams params_of(const EmberRaggedBatch &b, int slots) {
    SpanParams p{};
    p.q = b.q, p.k = b.k_cache, p.v = b.v_cache, p.out = b.out;
    p.query_start = b.query_start, p.positions = b.positions, p.tables = b.block_tables;
    p.q_stride = b.q_stride;
    p.T = b.T, p.S = b.S, p.max_blocks = b.max_blocks, p.n_heads = b.n_heads, p.n_kv = b.n_kv;
    p.G = b.n_heads / b.n_kv, p.num_blocks = b.num_blocks, p.slots = slots;
    p.part_acc = static_cast<float *>(b.workspace);
    if (p.part_acc) p.part_ml = p.part_acc + static_cast<int64_t>(b.T) * b.n_heads * slots * kHeadDim;
    p.window = kNoWindow;
    p.scale_log2 = b.scale * kLog2e;
    return p;
}

template <typename T>
hipError_t run(const SpanParams &p, const Launch &l, hipStream_t stream) {
    const int64_t first = groups_of(l.first, p.n_kv), second = l.second.units ? groups_of(l.second, p.n_kv) : 0;
    if (l.first_tiled) {
        if constexpr (sizeof(T) == 2) {
            if (first) hipLaunchKernelGGL(span_tile_kernel, dim3(static_cast<unsigned>(first)), dim3(kThreads), 0, stream, p, l.first);
            if (second)
                hipLaunchKernelGGL(span_walk_kernel<T>, dim3(static_cast<unsigned>(second)), dim3(kThreads), 0, stream, p,
                                   l.second, l.second, static_cast<int>(second));
        }
    } else if (first + second) {
        hipLaunchKernelGGL(span_walk_kernel<T>, dim3(static_cast<unsigned>(first + second)), dim3(kThreads), 0, stream, p,
                           l.first, l.second, static_cast<int>(first));
    }
    if (l.slots > 1) {
        const int64_t rows = static_cast<int64_t>(p.T) * p.n_heads;
        hipLaunchKernelGGL(span_merge_kernel<T>, dim3(static_cast<unsigned>((rows + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, p);
    }
    return hipGetLastError();
}

// The launch that the workspace has room for.
template <typename Plan>
int fit(const char *who, const EmberRaggedBatch &b, Plan plan, Launch &l) {
    const int64_t room = b.workspace ? b.workspace_bytes : 0;
    for (int spread = 0; spread <= kLeastSpread; spread++) {
        l = plan(spread);
        if (partial_bytes(b, l.slots) <= room) break;
        if (spread == kLeastSpread)
            return set_error(EMBER_ERR_INVALID, "%s: needs %lld bytes of workspace at least (got %lld)", who,
                             static_cast<long long>(partial_bytes(b, l.slots)), static_cast<long long>(room));
    }
    if (groups_of(l.first, b.n_kv) + groups_of(l.second, b.n_kv) > INT_MAX)
        return set_error(EMBER_ERR_INVALID, "%s: too many work-groups for one launch", who);
    return EMBER_OK;
}

}  // namespace

int64_t window_workspace_bytes(const EmberWindowAttnArgs &a) { return partial_bytes(a.batch, plan_window(a, 0).most_slots); }
int64_t shared_prefix_workspace_bytes(const EmberPrefixAttnArgs &a) { return partial_bytes(a.batch, plan_prefix(a, 0).most_slots); }

int launch_window_attn(const EmberWindowAttnArgs &a, hipStream_t stream) {
    Launch l;
    if (int e = fit("window_attn", a.batch, [&](int spread) { return plan_window(a, spread); }, l)) return e;
    SpanParams p = params_of(a.batch, l.slots);
    p.window = a.window, p.sinks = a.sinks;
    return hip_status(a.batch.dtype == EMBER_DTYPE_F16 ? run<f16>(p, l, stream) : run<float>(p, l, stream), "window_attn");
}

int launch_shared_prefix_attn(const EmberPrefixAttnArgs &a, hipStream_t stream) {
    Launch l;
    if (int e = fit("shared_prefix_attn", a.batch, [&](int spread) { return plan_prefix(a, spread); }, l)) return e;
    SpanParams p = params_of(a.batch, l.slots);
    p.group_start = a.group_start, p.prefix_len = a.prefix_len, p.n_groups = a.n_groups;
    return hip_status(a.batch.dtype == EMBER_DTYPE_F16 ? run<f16>(p, l, stream) : run<float>(p, l, stream), "shared_prefix_attn");
}

}  // namespace ember::hip
