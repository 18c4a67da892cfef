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
// of the table is followed and a split is a run of virtual pages. Partials
// (running max, sum, unnormalised output) of rows that are split, over a long
// axis or into prefix and own keys, go to slots of the workspace, and a merge
// launch joins them in slot order: no atomics, the same bits every time.
//
// Two forms. Few rows (16 at most: decode, verify) are bound by the read of
// the pages: span_walk_kernel gives each wave pages of its own, straight from
// HBM. Many rows (prompt chunks, a group's rows before a long prefix) are bound by
// the products: span_tile_kernel shares 64-key blocks in LDS between waves of
// 32 rows each. span_mixed_kernel runs both in one launch.
//
// Measured (us a call among others, one MI355X; each kernel's own figures stand beside it):
//   walk   32 decodes, windows of 4096 tokens, 16 / 8 heads   75.4, 6.4 TB/s
//          64 verify runs of up to 5 tokens, windows of 1000  43.5, 6.1 TB/s
//          1 decode, a window of 512                           7.7: a chain of four trips to memory
//   tile   2000 tokens, windows of 4096                       86 to 89 (by the clock that a box settles at), 760 to 780 TFLOP/s
//   mixed  64 decodes behind 8000 shared tokens               55, of which the merge takes 5
//          256 decodes in 16 groups                          110 (4.7 TB/s), of which the merge takes 5
#include <algorithm>
#include <climits>

#include "capi_errors.hpp"
#include "device.hpp"
#include "kernels.hpp"
#include "paged_device.hpp"

namespace ember::hip {
namespace {

constexpr int kWalkRows = 16;              // query rows of a walk work-group: one MFMA column each
constexpr int kTileWaves = 4;              // a tile's waves in one key group: 32 query rows each
constexpr int kTileRows = 32 * kTileWaves;
constexpr int kTileThreads = kTileWaves * kWave;
constexpr int kBlockPages = 4;             // pages of a tile's key block
constexpr int kBlockKeys = kBlockPages * kPage;
static_assert(kBlockPages == kTileWaves);  // a wave loads one of them
constexpr uint32_t kNoWindow = 1u << 31;  // past any distance of two positions

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
    float *part_acc, *part_ml;  // [part_tokens, n_heads, slots][128], [part_tokens, n_heads, slots][2]
    int64_t q_stride;
    int T, S, max_blocks, n_heads, n_kv, G, num_blocks, n_groups, sinks, slots, part_tokens;
    uint32_t window;
    float scale_log2;
};

__device__ __forceinline__ int clamped(int x, int most) { return min(max(x, 0), most); }

// The rows of one work item and the bounds of the keys they see.
struct Rows {
    int t0, rows;     // first token, (token, head) rows
    int seq;          // the table's row
    int base, limit;  // keys base .. limit - 1
    int pos;          // the first token's position, if there is one token (rows == G)
    bool partial;     // whether the step is split (else the first split does all)
    int part0;        // the token of the workspace's first row
};

// The group of sequence s by 64-ary search (one step for up to 63 groups): whether it is in one, and its prefix length.
__device__ __forceinline__ bool group_of(const SpanParams &p, int s, int lane, int &prefix) {
    int lo = 0, n = p.n_groups;  // the group, if there is one, is among lo .. lo + n - 1
    prefix = 0;
    while (n > 0) {
        const int step = (n + kWave - 2) / (kWave - 1);  // lanes 0 .. 62 look at a start each, the one behind them at the end
        const int at = min(lo + lane * step, p.n_groups);
        const int start = p.group_start[at], len = p.prefix_len[min(at, p.n_groups - 1)];
        const int c = __popcll(__builtin_amdgcn_ballot_w64(lane * step < n && start <= s));  // starts ascend: lanes 0 .. c - 1
        if (c == 0) return false;
        if (step == 1) {
            prefix = max(0, __builtin_amdgcn_readlane(len, c - 1));
            const bool in = s < __builtin_amdgcn_readlane(start, c);
            prefix = in ? prefix : 0;
            return in;
        }
        const int from = lo + (c - 1) * step;
        n = min(step, lo + n - from);
        lo = from;
    }
    return false;
}

// What one trip to memory can tell of a work item. A sequence of a pure decode step has its token at row `unit`: its
// position is requested beside query_start and used if query_start says so.
__device__ __forceinline__ Rows rows_of(const SpanParams &p, const Phase &ph, int unit, int lane, bool &grouped) {
    Rows r;
    int s0 = unit, s1 = unit + 1;
    r.base = 0;
    r.limit = INT_MAX;
    grouped = true;
    if (ph.kind == kPrefixRows) {
        s0 = uniform_load(p.group_start + unit);
        s1 = uniform_load(p.group_start + unit + 1);
        r.limit = max(0, uniform_load(p.prefix_len + unit));
        s0 = clamped(s0, p.S);
        s1 = max(clamped(s1, p.S), s0);
    }
    int guess = uniform_load(p.positions + min(unit, p.T - 1));
    const int t0 = uniform_load(p.query_start + s0), t1 = uniform_load(p.query_start + s1);
    if (ph.kind == kOwnRows) grouped = group_of(p, unit, lane, r.base);
    // A step of more tokens than the workspace has rows for (more than the sizes named) is not split.
    int least = 0, most = p.T;
    r.partial = p.slots > 1;
    r.part0 = 0;
    if (r.partial && p.part_tokens < p.T) {
        r.part0 = clamped(uniform_load(p.query_start), p.T);
        r.partial = clamped(uniform_load(p.query_start + p.S), p.T) - r.part0 <= p.part_tokens;
        if (r.partial) least = r.part0, most = min(r.part0 + p.part_tokens, p.T);
    }
    r.t0 = min(max(t0, least), most);
    r.rows = max(0, min(t1, most) - r.t0) * p.G;
    r.seq = min(s0, p.S - 1);
    if (r.rows == p.G && r.t0 != unit) guess = uniform_load(p.positions + r.t0);
    r.pos = guess;
    return r;
}

// The virtual pages of rows at positions min_pos .. max_pos whose highest visible keys are at most max_top.
struct Span {
    int lo;       // the first key that a window reaches
    int head;     // virtual pages 0 .. head - 1 are the table's first ones; page v >= head is the table's v + skip
    int skip, pages;
    __device__ __forceinline__ int page(int v) const { return v < head ? v : v + skip; }
};

// The first key that a window reaches from a position.
__device__ __forceinline__ int window_start(int pos, uint32_t window) {
    return window == kNoWindow ? 0 : pos - static_cast<int>(window) + 1;
}

__device__ __forceinline__ Span span_of(const Rows &r, uint32_t window, int sinks, int min_pos, int max_top) {
    Span s;
    // A window that starts behind the last key has none: it starts there at most (the end of a page, if there are first
    // tokens), so that no page number is further than the table's end and a tile's blocks behind it.
    s.lo = min(max(max(r.base, window_start(min_pos, window)), 0), max_top + 1);
    const int first = s.lo / kPage;
    s.head = min((max(min(sinks, max_top + 1), 0) + kPage - 1) / kPage, first);
    s.skip = first - s.head;
    s.pages = s.head + (s.lo <= max_top ? max_top / kPage - first + 1 : 0);
    return s;
}

// Whether every key of a page is visible to every row (positions min_pos .. max_pos, highest keys at least min_top).
__device__ __forceinline__ bool whole_page(int page, const Rows &r, uint32_t window, int sinks, int max_pos, int min_top) {
    const int j0 = page * kPage;
    return j0 >= r.base && j0 + kPage - 1 <= min_top && (static_cast<uint32_t>(max_pos - j0) < window || j0 + kPage <= sinks);
}

__device__ __forceinline__ bool visible(int j, int base, int top, int pos, uint32_t window, int sinks) {
    return j >= base && j <= top && (static_cast<uint32_t>(pos - j) < window || j < sinks);
}

// ---- few rows: a page per wave ----

// Lane l = 16 g + c serves query column c, the item's row c (columns past the last repeat it). f16 pages: S^T = K Q^T
// on v_mfma_f32_16x16x32_f16 (step s takes dims 32 s + 8 g .. + 7), O^T += V^T P^T on v_mfma_f32_16x16x16_f16. f32
// pages use v_mfma_f32_16x16x4_f32 the same way: step s of the scores takes dim 16 (s / 4) + 4 g + s % 4 from lane
// group g, so a lane loads key c in 16-byte pieces; step v of the values takes key 4 g + v, which the lane's own
// scores belong to. Keys of the f16 form pass through LDS (direct loads of four whole rows an instruction, swizzled).
// Where a CU runs 16 waves, each has half a page in flight; DEEP keeps two whole pages instead, for 8 waves a CU.
//
// Bound by HBM where the launch fills the chip (6.4 TB/s), else by latency: query_start and positions, the table, the
// pages, the merge of the waves are trips that wait for one another, 8 us for one page a wave. Hence a page per wave
// (a work-group per kv head reads 16 pages at once), W = 16 waves up to one work-group a CU, 8 up to two, 4 beyond,
// no scratch (any spill costs a launch 7 to 10 us), and lane offsets that go into the loads' immediates.
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

constexpr int kWalkRowPitch = kHeadDim + 4;               // floats of a row's partial: 16 rows' pieces of one dim on distinct banks
constexpr int kWalkWave = kWalkRows * kWalkRowPitch;      // floats of a wave's region (f16: it also stages keys, 4 KiB a page)
constexpr int kStageWords = kPage * kHeadDim / 2;
constexpr int walk_lds_floats(int W) { return W * (kWalkWave + 2 * kWalkRows); }

template <typename T, int W, bool DEEP>  // W waves
__device__ __forceinline__ void walk_item(const SpanParams &p, const Phase &ph, const int id, float *red) {
    constexpr int D = kHeadDim, kThreads = W * kWave, RP = kWalkRowPitch, RW = kWalkWave;
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int KQ = F16 ? 4 : 8;  // 16-byte pieces of a row of q or K in a lane
    float *const red_m = red + W * RW, *const red_l = red_m + W * kWalkRows;  // [row][wave]
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int g = lane >> 4, c = lane & 15;
    const int kvh = id % p.n_kv;
    int rest = id / p.n_kv;
    const int tile0 = rest % ph.tiles;
    rest /= ph.tiles;
    const int split = rest % ph.splits, unit = rest / ph.splits;

    // Up to its pages a work-group runs at raised wave priority: the CU's streaming waves otherwise win the issue
    // arbitration, and its few dependent loads wait behind theirs.
    __builtin_amdgcn_s_setprio(3);
    bool grouped;
    const Rows r = rows_of(p, ph, unit, lane, grouped);
    const int32_t *const table = p.tables + static_cast<int64_t>(r.seq) * p.max_blocks;
    const int64_t head_off = static_cast<int64_t>(kvh) * (kPage * D), block_stride = static_cast<int64_t>(p.n_kv) * (kPage * D);
    const T *const kbase = static_cast<const T *>(p.k) + head_off, *const vbase = static_cast<const T *>(p.v) + head_off;
    const uint32_t window = ph.kind == kWindowRows ? p.window : kNoWindow;
    const int sinks = ph.kind == kWindowRows ? p.sinks : 0;
    const int table_top = p.max_blocks * kPage - 1;
    const bool partial = r.partial;
    if (!partial && split > 0) return;
    // Without a window the pages start at the base: their ids are requested before the positions are known.
    const int early_page = r.base / kPage + split * ph.pages + wave + lane * W;
    int early = -1;
    if (ph.kind != kWindowRows && early_page < p.max_blocks) early = table[early_page];

    for (int row0 = tile0 * kWalkRows; row0 < r.rows; row0 += ph.tiles * kWalkRows) {
        const int nrows = min(kWalkRows, r.rows - row0);
        const int my_row = row0 + min(c, nrows - 1);
        const int my_tok = r.t0 + my_row / p.G, my_head = kvh * p.G + my_row % p.G;
        auto top_of = [&](int pos) { return min(min(pos, r.limit - 1), table_top); };
        int my_pos, min_pos, max_pos, min_top, max_top;
        if (r.rows == p.G) {
            my_pos = min_pos = max_pos = max(r.pos, -1);
            min_top = max_top = top_of(my_pos);
        } else {
            my_pos = max(p.positions[my_tok], -1);
            min_pos = max_pos = my_pos;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                min_pos = min(min_pos, __shfl_xor(min_pos, o, kWave));
                max_pos = max(max_pos, __shfl_xor(max_pos, o, kWave));
            }
            min_pos = uniform(min_pos), max_pos = uniform(max_pos);
            min_top = top_of(min_pos), max_top = top_of(max_pos);
        }
        const int my_top = top_of(my_pos);
        u32x4 qf[KQ];  // the row's q as the scores' B operand
        {
            const T *qp = static_cast<const T *>(p.q) + my_tok * p.q_stride + my_head * D;
#pragma unroll
            for (int i = 0; i < KQ; i++) qf[i] = *reinterpret_cast<const u32x4 *>(qp + (F16 ? 32 * i + 8 * g : 16 * i + 4 * g));
        }
        const Span sp = span_of(r, window, sinks, min_pos, max_top);
        const int v0 = min(split * ph.pages, sp.pages);
        const int v1 = split == ph.splits - 1 || !partial ? sp.pages : min(v0 + ph.pages, sp.pages);
        if (partial && v0 >= v1) {  // nothing to read: the slot is empty
            if (tid < nrows) {
                const int64_t at = static_cast<int64_t>(r.t0 - r.part0 + (row0 + tid) / p.G) * p.n_heads + kvh * p.G + (row0 + tid) % p.G;
                float2 *const ml = reinterpret_cast<float2 *>(p.part_ml) + at * p.slots;
                ml[ph.slot0 + split] = make_float2(kNoKeys, 0.0f);
                if (!grouped && split == 0)
                    for (int i = 0; i < ph.slot0; i++) ml[i] = make_float2(kNoKeys, 0.0f);
            }
            continue;
        }

        float mc = kNoKeys, lc = 0.0f;
        f32x4 o[8];  // o[t][v]: dim 32 g + 8 v + t of column c
#pragma unroll
        for (int t = 0; t < 8; t++) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t *const kstage = reinterpret_cast<uint32_t *>(&red[wave * RW]);
        // The swizzled stage: slot 16 k + (q ^ k) holds chunk q of key k. Load i writes keys 4 i .. + 3 (lane l the 16
        // bytes at 16 l), step i reads chunk 4 i + g of key c; both differ between i by an exclusive or and a constant.
        const uint32_t k_dma = 256u * g + 16u * (c ^ g), k_rd = 256u * c + 16u * (c ^ g);  // bytes
        const uint32_t v_off = F16 ? 1024u * g + 16u * c : 2048u * g + 32u * c, k_off = (F16 ? 256u : 512u) * c + 16u * g;
        // Wave w takes pages w, w + W, ...; the block ids of up to 64 of them at a time, one a lane.
        for (int cv = v0 + wave; cv < v1; cv += W * kWave) {
            const int n = min(kWave, (v1 - cv + W - 1) / W);
            int ids = early;
            if (ph.kind == kWindowRows || cv != v0 + wave) ids = lane < n ? table[sp.page(cv + lane * W)] : -1;
            using Page = WalkPage<T>;
            auto desc_of = [&](const T *base, int j) {
                const int blk = __builtin_amdgcn_readlane(ids, min(j, n - 1));
                const bool live = j < n && blk >= 0 && blk < p.num_blocks;  // dead: no records, the loads give zeros
                return __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base) + (live ? blk : 0) * block_stride, 0,
                                                         live ? kPage * D * static_cast<int>(sizeof(T)) : 0, kDescWord3);
            };
            // A lane's offsets are made opaque where they are used: their constant parts then go into the loads, where
            // the compiler would hold each sum in a register of its own across the loop.
            auto here = [](uint32_t x) {
                asm volatile("" : "+v"(x));
                return x;
            };
            auto fetch_keys = [&](Page &A, int j, int buffer) {
                const __amdgpu_buffer_rsrc_t d = desc_of(kbase, j);
                const uint32_t off = here(F16 ? k_dma : k_off);
                if constexpr (F16) {
                    uint32_t *const to = kstage + buffer * kStageWords;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(
                            d, (__attribute__((address_space(3))) void *)(to + 256 * i), 16, (off ^ (64u * i)) + 1024u * i, 0, 0,
                            kNonTemporal);
                } else {
#pragma unroll
                    for (int i = 0; i < KQ; i++) A.k[i] = load_desc(d, off + 64u * i);
                }
            };
            auto fetch_values = [&](Page &A, int j) {
                const __amdgpu_buffer_rsrc_t d = desc_of(vbase, j);
                const uint32_t off = here(v_off);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (F16) {
                        A.v[i] = load_desc(d, off + 256u * i);
                    } else {
                        A.v[i][0] = load_desc(d, off + 512u * i);
                        A.v[i][1] = load_desc(d, off + 512u * i + 16u);
                    }
                }
            };
            // Page j: its scores and the online softmax, then its values; `next` is called between, once its keys
            // have been read.
            auto consume = [&](Page &A, int j, int buffer, auto next) {
                const int page = sp.page(cv + j * W);
                f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};  // s[v]: raw score of key 4 g + v
                if constexpr (F16) {
                    // Loads end in order, and only so many are out behind the page's keys: its values, and DEEP the next
                    // page's keys and values.
                    if constexpr (DEEP) asm volatile("s_waitcnt vmcnt(12)" ::: "memory");
                    else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
                    __builtin_amdgcn_sched_barrier(0);
                    u32x4 kf[4];
                    const uint32_t off = here(k_rd);
                    const char *const from = reinterpret_cast<const char *>(kstage + buffer * kStageWords);
#pragma unroll
                    for (int i = 0; i < 4; i++) kf[i] = *reinterpret_cast<const u32x4 *>(from + (off ^ (64u * i)));
#pragma unroll
                    for (int i = 0; i < 4; i++) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(kf[i]), as_f16x8(qf[i]), s, 0, 0, 0);
                } else {
                    f32x4 s2 = s;  // two chains: each product waits for the one before it
#pragma unroll
                    for (int i = 0; i < KQ; i++)
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(A.k[i][e]), __uint_as_float(qf[i][e]), s, 0, 0, 0);
                            s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(A.k[i][e + 1]), __uint_as_float(qf[i][e + 1]), s2, 0, 0, 0);
                        }
                    s = s + s2;
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
                const float top = groups_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))) * p.scale_log2;
                const float mn = fmaxf(mc, F16 ? below(top, kMostExponent) : top);
                const float corr = exp2_hw(mc - mn);
                mc = mn;
                float mul = p.scale_log2, add = -mn;
                if (const bool far = fabsf(mn) >= kFar; __builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
                    for (int v = 0; v < 4; v++) s[v] = far ? s[v] * mul + add : __builtin_fmaf(s[v], mul, add);
                    mul = 1.0f, add = 0.0f;
                }
                float w[4];
#pragma unroll
                for (int v = 0; v < 4; v++) w[v] = exp2_hw(__builtin_fmaf(s[v], mul, add));
                // f16: the weights are rounded to f16, the products' operand, and summed as rounded, so that the
                // rounding of a weight moves numerator and denominator alike: 2^-11 of it at most down to 2^-29 of
                // the largest, 2^-40 of the largest below.
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
                next();
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
            };
            // Keys and values are requested in the order that the waits count on: nothing moves across the fences.
            auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
            auto fetch = [&](Page &A, int j, int buffer) {
                fence();
                fetch_keys(A, j, buffer);
                fence();
                fetch_values(A, j);
                fence();
            };
            if constexpr (DEEP) {
                static_assert(2 * kStageWords <= kWalkWave);
                Page A, B;
                fetch(A, 0, 0);
                fetch(B, 1, 1);
                __builtin_amdgcn_s_setprio(0);
                for (int j = 0; j < n; j += 2) {
                    consume(A, j, 0, fence);
                    fetch(A, j + 2, 0);
                    if (j + 1 < n) consume(B, j + 1, 1, fence);
                    fetch(B, j + 3, 1);
                }
            } else {
                Page A;
                fetch(A, 0, 0);
                __builtin_amdgcn_s_setprio(0);
                for (int j = 0; j < n; j++) {
                    consume(A, j, 0, [&] {
                        fence();
                        fetch_keys(A, j + 1, 0);
                        fence();
                    });
                    fence();
                    fetch_values(A, j + 1);
                    fence();
                }
            }
            // The fetches past the last page still write zeros into the stage, where the next chunk's keys or the
            // wave's partial go.
            if constexpr (F16) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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
                red_m[c * W + wave] = mc;
                red_l[c * W + wave] = lc;
            }
        }
        __syncthreads();
        for (int i = tid; i < nrows * (D / 2); i += kThreads) {
            const int row = i / (D / 2), d = 2 * (i % (D / 2));
            float M = kNoKeys, L = 0.0f;
#pragma unroll 4
            for (int w = 0; w < W; w++) M = fmaxf(M, red_m[row * W + w]);
            float2 O = make_float2(0.0f, 0.0f);
#pragma unroll 4
            for (int w = 0; w < W; w++) {
                const float f = exp2_hw(red_m[row * W + w] - M);
                const float2 x = *reinterpret_cast<const float2 *>(&red[w * RW + row * RP + d]);
                L = L + red_l[row * W + w] * f;
                O.x = O.x + x.x * f;
                O.y = O.y + x.y * f;
            }
            const int64_t at = static_cast<int64_t>(r.t0 - (partial ? r.part0 : 0) + (row0 + row) / p.G) * p.n_heads + kvh * p.G + (row0 + row) % p.G;
            if (partial) {
                const int64_t slot = at * p.slots + ph.slot0 + split;
                float2 *const ml = reinterpret_cast<float2 *>(p.part_ml);
                *reinterpret_cast<float2 *>(p.part_acc + slot * D + d) = O;
                if (d == 0) {
                    ml[slot] = make_float2(M, L);
                    if (!grouped && split == 0)  // a row of no group: its prefix slots hold nothing
                        for (int k = 0; k < ph.slot0; k++) ml[at * p.slots + k] = make_float2(kNoKeys, 0.0f);
                }
            } else {
                T *const dst = static_cast<T *>(p.out) + at * D + d;
                dst[0] = from_f32<T>(filled(L) ? O.x / L : 0.0f);
                dst[1] = from_f32<T>(filled(L) ? O.y / L : 0.0f);
            }
        }
        __syncthreads();  // the regions are the next row tile's stages
    }
}

// Two phases in one launch (b.units may be 0). A CU holds 16 waves of the f16 form and 8 of the f32 form.
template <typename T, int W>
__global__ void __launch_bounds__(W *kWave, (sizeof(T) == 2 ? 4 : 2))
    span_walk_kernel(SpanParams p, Phase a, Phase b, int a_groups) {
    __shared__ __align__(16) float red[walk_lds_floats(W)];
    const int id = static_cast<int>(blockIdx.x);
    const bool second = id >= a_groups;
    walk_item<T, W, false>(p, second ? b : a, second ? id - a_groups : id, red);
}

// ---- many rows: key blocks shared in LDS (f16) ----

// Wave w owns rows 32 w .. 32 w + 31 of the tile; lane l = 32 h + c serves row c.
//   S^T = K Q^T   v_mfma_f32_32x32x16_f16: lane l ends with row c's scores of keys 8 (i / 4) + 4 h + i % 4 of each
//                 32-key half, i = 0 .. 15, so a row lives in two lanes: its max and sum meet through one
//                 v_permlane32_swap, and rescaling O touches no other lane.
//   O^T += V^T P^T  the lane's scores, as weights in f16, are the B operand as they stand (the order of the keys
//                 inside one product is free); the A operand, the same keys of dim c, comes from the transposing
//                 LDS read: lane r of a 16-lane block reads four dims of key r / 4, lane i receives dim i of 4 keys.
// LDS rows, halves. Keys: 68 dwords, so that 16 rows' pieces of 16 bytes, read at once, lie on the 64 banks side by side.
// Values: 80 dwords, so that the four rows and two dim blocks of a transposing read of 32 lanes do.
constexpr int kKeyRow = kHeadDim + 8, kValueRow = kHeadDim + 32;
typedef __fp16 tr16x4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __attribute__((address_space(3))) tr16x4 lds_tr16x4;

constexpr int kAhead = 4;  // value operands in flight ahead of their products

// Bound by the two waves of a SIMD taking turns: at 2000 tokens behind 12,000 (windows of 4096) the matrix unit is
// busy 34% of the cycles, the VALU 35%, LDS 26%, HBM hardly at all. 128 rows share a block's 32 KiB, and a page a wave
// is loaded a block ahead through registers. Tried: loads straight to LDS with three key buffers, and the groups half a
// step apart (4 us less, for twice the code), weights of the next keys between the products of the last (2 us more),
// 8 value operands ahead in place of 4 (no change).
//
// KG key groups of 4 waves, the same rows each: group g takes blocks g, g + KG, ... through buffers of its own, and
// the last ones hand their partials to group 0 through LDS.
constexpr int kKeyBuffer = kBlockKeys * kKeyRow, kValueBuffer = kBlockKeys * kValueRow;
constexpr int tile_lds_bytes(int KG) { return KG * 2 * (kKeyBuffer + kValueBuffer) * static_cast<int>(sizeof(f16)) + 64; }

template <int KG>
__device__ __forceinline__ void tile_item(const SpanParams &p, const Phase &ph, const int id, unsigned char *lds) {
    constexpr int D = kHeadDim;
    f16 *const k_all = reinterpret_cast<f16 *>(lds), *const v_all = k_all + KG * 2 * kKeyBuffer;
    int *const ext = reinterpret_cast<int *>(v_all + KG * 2 * kValueBuffer);  // [wave][2]
    const int group = KG == 1 ? 0 : uniform(static_cast<int>(threadIdx.x) / kTileThreads);
    const int tid = static_cast<int>(threadIdx.x) % kTileThreads, lane = tid % kWave, wave = uniform(tid / kWave);
    f16 *const k_lds = k_all + group * 2 * kKeyBuffer, *const v_lds = v_all + group * 2 * kValueBuffer;  // two buffers each
    const int h = lane >> 5, c = lane & 31;
    const int kvh = id % p.n_kv;
    int rest = id / p.n_kv;
    const int tile0 = rest % ph.tiles;
    rest /= ph.tiles;
    const int split = rest % ph.splits, unit = rest / ph.splits;

    // Up to its pages a work-group runs at raised wave priority: the CU's streaming waves otherwise win the issue
    // arbitration, and its few dependent loads wait behind theirs.
    __builtin_amdgcn_s_setprio(3);
    bool grouped;
    const Rows r = rows_of(p, ph, unit, lane, grouped);
    const bool partial = r.partial;
    if (!partial && split > 0) return;
    const int32_t *const table = p.tables + static_cast<int64_t>(r.seq) * p.max_blocks;
    const int64_t head_off = static_cast<int64_t>(kvh) * (kPage * D), block_stride = static_cast<int64_t>(p.n_kv) * (kPage * D);
    const f16 *const kbase = static_cast<const f16 *>(p.k) + head_off, *const vbase = static_cast<const f16 *>(p.v) + head_off;
    const uint32_t window = ph.kind == kWindowRows ? p.window : kNoWindow;
    const int sinks = ph.kind == kWindowRows ? p.sinks : 0;

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
        if (group == 0 && lane == 0) ext[2 * wave] = lo_pos, ext[2 * wave + 1] = hi_top;
        __syncthreads();
        int min_pos = lo_pos, max_top = hi_top;  // of the tile
#pragma unroll
        for (int w = 0; w < kTileWaves; w++) min_pos = min(min_pos, ext[2 * w]), max_top = max(max_top, ext[2 * w + 1]);
        min_pos = uniform(min_pos), max_top = uniform(max_top);
        const Span sp = span_of(r, window, sinks, min_pos, max_top);
        const int v0 = min(split * ph.pages, sp.pages);
        const int v1 = split == ph.splits - 1 || !partial ? sp.pages : min(v0 + ph.pages, sp.pages);
        const int blocks = (v1 - v0 + kBlockPages - 1) / kBlockPages;  // this group's: group, group + KG, ...

        // This lane's part of a value operand: key 4 h + r / 4, dims 16 (l / 16 % 2) + 4 (r % 4) .. + 3 of its 16-lane block.
        const int v_at = (4 * h + lane % 16 / 4) * kValueRow + 16 * (lane / 16 % 2) + 4 * (lane % 4);
        float m = -INFINITY, l = 0.0f;
        f32x16 o[4];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] = 0.0f;

        // Keys that this lane's row sees: n from `from` on, and those below `sink_end`.
        const int from = max(r.base, max(window_start(my_pos, window), 0));
        const uint32_t n_from = max(my_top - from + 1, 0);
        const int sink_end = min(sinks, my_top + 1);
        // Virtual pages whole0 .. whole1 - 1: every row of the wave sees every key of them.
        const int whole_key = max(r.base, window_start(hi_pos, window));
        const int whole0 = static_cast<int>((static_cast<uint32_t>(max(whole_key, 0)) + kPage - 1) / kPage) - sp.skip;
        const int whole1 = (lo_top + 1) / kPage - sp.skip;
        // Keys that some row of the tile sees, likewise. Others may hold anything: their values are read as zeros
        // (an offset past the page's records), so that a zero weight meets no NaN.
        const uint32_t n_live = max(max_top - sp.lo + 1, 0);
        const int sink_live = min(sinks, max_top + 1);

        // A block's pages into registers, a page a wave: 16 bytes of keys 4 i + l / 16 a lane. The ids of 64 steps' pages
        // are held one a lane; one outside the pool has no records, and its loads give zeros.
        u32x4 kr[4], vr[4];
        // Step b of this group reads virtual pages first_page(b) .. + 3.
        auto first_page = [&](int b) { return v0 + (b * KG + group) * kBlockPages; };
        auto id_of = [&](int b) {
            const int v = first_page(b) + wave;
            return v < v1 ? table[sp.page(v)] : -1;
        };
        int ids = -1, next_ids = id_of(lane);
        // Lane offsets are made opaque: their constant parts then go into the accesses, where the compiler would hold
        // each sum in a register of its own across the loop.
        auto here = [](int x) {
            asm volatile("" : "+v"(x));
            return x;
        };
        auto fetch = [&](int b) {
            if (b % kWave == 0) {
                ids = next_ids;
                next_ids = id_of(b + kWave + lane);
            }
            const int blk = __builtin_amdgcn_readlane(ids, b % kWave);
            const bool live = blk >= 0 && blk < p.num_blocks;
            const int64_t at = (live ? blk : 0) * block_stride;
            const int bytes = live ? kPage * D * static_cast<int>(sizeof(f16)) : 0;
            const __amdgpu_buffer_rsrc_t kd = __builtin_amdgcn_make_buffer_rsrc(const_cast<f16 *>(kbase) + at, 0, bytes, kDescWord3);
            const __amdgpu_buffer_rsrc_t vd = __builtin_amdgcn_make_buffer_rsrc(const_cast<f16 *>(vbase) + at, 0, bytes, kDescWord3);
            auto load = [](__amdgpu_buffer_rsrc_t d, int off) {
                return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(d, off, 0, 0));
            };
            constexpr int kPast = kPage * D * static_cast<int>(sizeof(f16));
            const int at_lane = here(lane), off = 16 * at_lane, key0 = sp.page(first_page(b) + wave) * kPage + at_lane / 16;
#pragma unroll
            for (int i = 0; i < 4; i++) kr[i] = load(kd, off + 1024 * i);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int key = key0 + 4 * i;
                const bool seen = (static_cast<uint32_t>(key - sp.lo) < n_live) | (key < sink_live);
                vr[i] = load(vd, seen ? off + 1024 * i : kPast);
            }
        };
        auto stage = [&](int b) {
            const int at_lane = here(lane), key = kPage * wave + at_lane / 16, dim = at_lane % 16 * 8;
            f16 *const kp = k_lds + (b & 1) * kKeyBuffer + key * kKeyRow + dim;
            f16 *const vp = v_lds + (b & 1) * kValueBuffer + key * kValueRow + dim;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                *reinterpret_cast<u32x4 *>(kp + 4 * i * kKeyRow) = kr[i];
                *reinterpret_cast<u32x4 *>(vp + 4 * i * kValueRow) = vr[i];
            }
        };
        const int steps = (blocks + KG - 1) / KG;
        if (steps > 0) {
            fetch(0);
            __builtin_amdgcn_s_setprio(0);
            stage(0);
        }
        __syncthreads();
        for (int b = 0; b < steps; b++) {
            if (b + 1 < steps) fetch(b + 1);
            const f16 *const kl = k_lds + (b & 1) * kKeyBuffer + c * kKeyRow + 8 * h;
            const f16 *const vl = v_lds + (b & 1) * kValueBuffer + v_at;
            // Scores: the operands of a 32-key half are all requested before its first product, and each is
            // replaced by the other half's as soon as its product is issued.
            f32x16 s[2];
            f16x8 ka[8];
#pragma unroll
            for (int i = 0; i < 8; i++) ka[i] = *reinterpret_cast<const f16x8 *>(kl + 16 * i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < 2; t++) {
#pragma unroll
                for (int i = 0; i < 16; i++) s[t][i] = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[i], qf[i], s[t], 0, 0, 0);
                    if (t == 0) ka[i] = *reinterpret_cast<const f16x8 *>(kl + 32 * kKeyRow + 16 * i);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            // The first values, in flight during the softmax: operand n = 4 j + t is dim tile t of keys 16 j .. + 15.
            auto value = [&](int n) {
                const f16 *const at = vl + n / 4 * 16 * kValueRow + n % 4 * 32;
                const f16x4 lo4 = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr16x4 *)at));
                const f16x4 hi4 = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr16x4 *)(at + 8 * kValueRow)));
                return f16x8{lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
            };
            f16x8 va[kAhead];
#pragma unroll
            for (int n = 0; n < kAhead; n++) va[n] = value(n);
            __builtin_amdgcn_sched_barrier(0);
            // (a run is whole blocks for every group, so pages past it lie past every row's keys)
            const int vb = first_page(b);
            if (!(vb >= whole0 && vb + kBlockPages <= whole1)) {
#pragma unroll
                for (int j = 0; j < kBlockPages; j++) {
                    const int key0 = sp.page(vb + j) * kPage + 4 * h;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int key = key0 + 8 * (i / 4) + i % 4;
                        const bool see = (static_cast<uint32_t>(key - from) < n_from) | (key < sink_end);
                        s[j / 2][8 * (j % 2) + i] = see ? s[j / 2][8 * (j % 2) + i] : -INFINITY;
                    }
                }
            }
            float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
            for (int i = 1; i < 16; i++) top = fmaxf(fmaxf(top, s[0][i]), s[1][i]);
            top = top * p.scale_log2;
            if (__builtin_amdgcn_ballot_w64(top - m > kMostExponent)) {
                const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                const float row_top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
                const bool grow = row_top - m > kMostExponent;
                const float reference = below(row_top, kMostExponent - kLazy);
                const float corr = grow ? exp2_hw(m - reference) : 1.0f;  // 0 from a row that had seen nothing
                m = grow ? reference : m;
                l = l * corr;
#pragma unroll
                for (int t = 0; t < 4; t++) o[t] = o[t] * corr;
            }
            float mul = p.scale_log2, neg = m == -INFINITY ? 0.0f : -m;
            if (const bool far = fabsf(neg) >= kFar; __builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[t][i] = far ? s[t][i] * mul + neg : __builtin_fmaf(s[t][i], mul, neg);
                mul = 1.0f, neg = 0.0f;
            }
            const f16x2 ones = {static_cast<f16>(1.0f), static_cast<f16>(1.0f)};
            f16x8 w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    w[j][i] = static_cast<f16>(exp2_hw(__builtin_fmaf(s[j / 2][8 * (j % 2) + i], mul, neg)));
#pragma unroll
                for (int i = 0; i < 4; i++) l = __builtin_amdgcn_fdot2(f16x2{w[j][2 * i], w[j][2 * i + 1]}, ones, l, false);
            }
#pragma unroll
            for (int n = 0; n < 16; n++) {
                o[n % 4] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[n % kAhead], w[n / 4], o[n % 4], 0, 0, 0);
                if (n + kAhead < 16) va[n % kAhead] = value(n + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (b + 1 < steps) stage(b + 1);
            __syncthreads();
        }

        if constexpr (KG == 2) {  // group 1's partial, through the buffers (every wave is past its last block)
            f32x4 *const hand = reinterpret_cast<f32x4 *>(k_all) + tid;
            static_assert(17 * kTileThreads * sizeof(f32x4) <= KG * 2 * kKeyBuffer * sizeof(f16));
            if (group == 1) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    hand[i * kTileThreads] = f32x4{o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1], o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]};
                hand[16 * kTileThreads] = f32x4{m, l, 0.0f, 0.0f};
            }
            __syncthreads();
            if (group == 0) {
                const f32x4 ml = hand[16 * kTileThreads];
                const float top = fmaxf(m, ml[0]);
                const float f0 = m == -INFINITY ? 0.0f : exp2_hw(m - top), f1 = ml[0] == -INFINITY ? 0.0f : exp2_hw(ml[0] - top);
                m = top;
                l = l * f0 + ml[1] * f1;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const f32x4 x = hand[i * kTileThreads];
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i / 4][4 * (i % 4) + e] = o[i / 4][4 * (i % 4) + e] * f0 + x[e] * f1;
                }
            }
            __syncthreads();  // the buffers are the next row tile's
        }
        if (group == 0 && mine) {
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
            l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
            const int64_t at = static_cast<int64_t>(my_tok - (partial ? r.part0 : 0)) * p.n_heads + my_head;
            if (partial) {
                const int64_t slot = at * p.slots + ph.slot0 + split;
                float *const dst = p.part_acc + slot * D + 4 * h;
                if (blocks > 0) {
#pragma unroll
                    for (int i = 0; i < 16; i++)  // dims 32 (i / 4) + 8 (i % 4) + 4 h .. + 3
                        *reinterpret_cast<float4 *>(dst + 8 * i) = make_float4(o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1],
                                                                               o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]);
                }
                if (h == 0) *reinterpret_cast<float2 *>(p.part_ml + slot * 2) = make_float2(filled(l) ? m : kNoKeys, l);
            } else {
                f16 *const dst = static_cast<f16 *>(p.out) + at * D + 4 * h;
                const float inv = filled(l) ? 1.0f / l : 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    f16x4 y;
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = static_cast<f16>(o[i / 4][4 * (i % 4) + e] * inv);
                    *reinterpret_cast<f16x4 *>(dst + 8 * i) = y;
                }
            }
        }
    }
}

template <int KG>
__global__ void __launch_bounds__(KG *kTileThreads, 2) span_tile_kernel(SpanParams p, Phase ph) {
    __shared__ __align__(16) unsigned char lds[tile_lds_bytes(KG)];
    tile_item<KG>(p, ph, static_cast<int>(blockIdx.x), lds);
}

// Tiles of a prefix beside walks of the own keys: the tiles are bound by their products, the walks by the memory, and
// a CU runs one work-group of each. 64 sequences on 8000 shared tokens (32 / 8 heads, 13 splits): tiles alone 31 us,
// walks alone 45, together 62, each with its launch and merge. The tiles come first: interleaved with the walks by 8
// work-groups they end later (68 us), and with raised priority for the walks too (65 us).
__global__ void __launch_bounds__(kTileThreads, 2) span_mixed_kernel(SpanParams p, Phase first, Phase walks, int tile_groups) {
    static_assert(tile_lds_bytes(1) >= walk_lds_floats(kTileWaves) * 4);
    __shared__ __align__(16) unsigned char lds[tile_lds_bytes(1)];
    const int id = static_cast<int>(blockIdx.x);
    if (id < tile_groups) tile_item<1>(p, first, id, lds);
    else walk_item<f16, kTileWaves, true>(p, walks, id - tile_groups, reinterpret_cast<float *>(lds));
}

// ---- the slots' merge: a wave per (token, head), two dims a lane ----
//
// 520 bytes a slot read, 3 to 5.5 us with the launch. A last-arriver's merge inside the launch before it (a count and
// device-scope stores) took longer than this launch.

constexpr int kMergeWaves = 4;

template <typename T>
__global__ void __launch_bounds__(kMergeWaves *kWave) span_merge_kernel(SpanParams p, int64_t first_row) {
    constexpr int D = kHeadDim, C = 8;  // slots whose partials are requested together
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    const int64_t at = first_row + static_cast<int64_t>(blockIdx.x) * kMergeWaves + uniform(static_cast<int>(threadIdx.x) / kWave);
    const int first = clamped(uniform_load(p.query_start), p.T), last = clamped(uniform_load(p.query_start + p.S), p.T);
    const int part0 = p.part_tokens < p.T ? first : 0;
    const int64_t tok = at / p.n_heads + part0;
    if (last - part0 > p.part_tokens || tok < first || tok >= last) return;  // not split, or of no sequence
    const float2 *const ml = reinterpret_cast<const float2 *>(p.part_ml) + at * p.slots;
    const float *const acc = p.part_acc + at * p.slots * D + 2 * lane;
    float M = kNoKeys, L = 0.0f, x = 0.0f, y = 0.0f;
    for (int s0 = 0; s0 < p.slots; s0 += kWave) {  // a lane holds a slot's (max, sum)
        const float2 mine = s0 + lane < p.slots ? ml[s0 + lane] : make_float2(kNoKeys, 0.0f);
        float top = mine.x;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
        top = fmaxf(M, top);
        const float corr = exp2_hw(M - top);
        M = top;
        L = L * corr, x = x * corr, y = y * corr;
        const float f = filled(mine.y) ? exp2_hw(mine.x - top) : 0.0f;
        const float l = mine.y * f;
        // Only slots that hold something are read (an empty one's partial is not written), C at a time.
        for (uint64_t left = __builtin_amdgcn_ballot_w64(filled(mine.y)); left != 0;) {
            float2 a[C];
            int slot[C];
            uint64_t rest = left;
#pragma unroll
            for (int i = 0; i < C; i++) {
                slot[i] = rest ? __builtin_ctzll(rest) : -1;
                a[i] = *reinterpret_cast<const float2 *>(acc + static_cast<int64_t>(s0 + max(slot[i], __builtin_ctzll(left))) * D);
                rest = rest & (rest - 1);
            }
            left = rest;
#pragma unroll
            for (int i = 0; i < C; i++) {
                const float w = slot[i] < 0 ? 0.0f : __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), max(slot[i], 0)));
                L = L + (slot[i] < 0 ? 0.0f : __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(l), max(slot[i], 0))));
                x = x + a[i].x * w;
                y = y + a[i].y * w;
            }
        }
    }
    T *const dst = static_cast<T *>(p.out) + (at + static_cast<int64_t>(part0) * p.n_heads) * D + 2 * lane;
    dst[0] = from_f32<T>(filled(L) ? x / L : 0.0f);
    dst[1] = from_f32<T>(filled(L) ? y / L : 0.0f);
}

// ---- host: phases and launches ----

struct Launch {
    Phase first{}, second{};  // second.units == 0: none
    bool tiled = false;       // the first phase is tiles
    int slots = 1, most_slots = 1;  // slots, and those that the workspace is sized for
    int pages = 0;                  // of a window's row tile, at most
    int tokens = 0;                 // that the workspace has room for
};

int64_t groups_of(const Phase &ph, int n_kv) { return static_cast<int64_t>(ph.units) * ph.tiles * ph.splits * n_kv; }

int64_t partial_bytes(const EmberRaggedBatch &b, int tokens, int slots) {
    return slots <= 1 ? 0 : static_cast<int64_t>(tokens) * b.n_heads * slots * (kHeadDim + 2) * static_cast<int64_t>(sizeof(float));
}

int tiles_for(int64_t tokens, int G, int rows) { return static_cast<int>(std::max<int64_t>(1, (tokens * G + rows - 1) / rows)); }

// `tokens` of every unit are the caller's longest run, or all of the step's: with many units most of the work-groups would
// find no rows, at about 1 us for 300 of them. Beyond kMostGroups a unit's row tiles share its work-groups, which also
// keeps a launch within HIP's 2^32 threads for any number of tokens. The share is odd: with an even one, 1000 decodes take
// 2 to 3 times as long, as if the few work-groups that have rows went to the same part of each XCD.
// Measured, us, at most 2^15, 2^16, 2^17 work-groups and without a bound: 1000 decodes without max_query, window 1724, 1748,
// 1763 and 4870, shared prefix 232, 275, 384 and 2012; 40 chunks of 512 tokens among 1000 sequences, shared prefix 1668,
// 1396, 1283 and 2124.
constexpr int64_t kMostGroups = 1 << 16;
constexpr int64_t kMostLaunch = UINT32_MAX / kTileThreads;  // work-groups of the launches that can be large: 256 threads

Phase rows_phase(int kind, int units, int64_t tokens, int G, int n_kv, bool tiled, int slot0) {
    const int64_t shared = (std::max<int64_t>(1, kMostGroups / (static_cast<int64_t>(units) * n_kv)) - 1) | 1;
    return Phase{kind, units, static_cast<int>(std::min<int64_t>(tiles_for(tokens, G, tiled ? kTileRows : kWalkRows), shared)), 1, 1, slot0};
}

// `spread` halves the work-groups asked for, step by step, until the workspace holds the partials.
constexpr int kLeastSpread = 10;  // no splits

// Cuts `pages` virtual pages into `runs` equal runs of a multiple of `unit`, or fewer where those reach the end sooner.
void set_runs(Phase &ph, int pages, int runs, int unit) {
    ph.pages = std::max(1, (pages + runs * unit - 1) / (runs * unit)) * unit;
    ph.splits = std::max(1, (pages + ph.pages - 1) / ph.pages);
}

// A window's work-group fills a CU (16 walking waves, 8 of f32 pages or of a tile), and with fewer work-groups than CUs
// the keys may be cut, at the price of the merge launch: the runs that take least by what a wave's page (a tile's pair
// of blocks) takes when the memory is not the bound, and a merge. One sequence, 8 kv heads, f16, measured: 2000 keys
// uncut 13.2 us, 4000 keys 25.6 us, of which 5 us are no page's; f32 3.3 us a page.
constexpr int kCus = 256;
constexpr double kMergeUs = 4.0;

int best_runs(int pages, int pages_a_step, double step_us, int most) {
    int best = 1;
    double least = 1e30;
    for (int runs = 1; runs <= most; runs++) {
        const int steps = (pages + runs * pages_a_step - 1) / (runs * pages_a_step);
        const double us = steps * step_us + (runs > 1 ? kMergeUs + 0.02 * runs : 0.0);
        if (us < least) least = us, best = runs;
    }
    return best;
}

Launch plan_window(const EmberWindowAttnArgs &a, int spread) {
    const EmberRaggedBatch &b = a.batch;
    const int G = b.n_heads / b.n_kv;
    const int64_t most = std::min(b.max_query, b.T);
    const bool f16_pages = b.dtype == EMBER_DTYPE_F16;
    Launch l;
    l.tokens = static_cast<int>(std::min<int64_t>(b.T, b.S * most));  // rows of padding need no partials
    l.tiled = f16_pages && most * G > kWalkRows;
    l.first = rows_phase(kWindowRows, b.S, most, G, b.n_kv, l.tiled, 0);
    // a tile's keys: the first tokens' pages, and the windows of its tokens
    const int64_t tokens = std::min<int64_t>(most, ((l.tiled ? kTileRows : kWalkRows) + G - 1) / G + 1);
    const int64_t near = (std::min<int64_t>(a.window, static_cast<int64_t>(b.max_blocks) * kPage) + tokens + kPage - 1) / kPage + 1;
    const int pages = static_cast<int>(std::min<int64_t>(b.max_blocks, near + (static_cast<int64_t>(a.sinks) + kPage - 1) / kPage));
    l.pages = pages;
    const int64_t items = static_cast<int64_t>(b.S) * l.first.tiles * b.n_kv;
    const int pages_a_step = l.tiled ? 2 * kBlockPages : f16_pages ? 16 : 8;
    l.most_slots = static_cast<int>(std::clamp<int64_t>((kCus >> spread) / items, 1, (pages + pages_a_step - 1) / pages_a_step));
    const int runs = best_runs(pages, pages_a_step, l.tiled ? 1.85 : f16_pages ? 1.2 : 3.3, l.most_slots);
    set_runs(l.first, pages, runs, l.tiled ? 2 * kBlockPages : 1);
    l.slots = l.first.splits;
    return l;
}

// A prefix's launch has a merge behind it in any case, so its walks are cut finely: two pages a wave or more.
constexpr int kWalkWant = 1024, kWalkFine = 8;

// Returns the runs that were allowed, which only grow with `pages` (the splits need not): the workspace is sized by them.
int cut_phase(Phase &ph, int n_kv, int pages, int least, int spread) {
    const int64_t items = static_cast<int64_t>(ph.units) * ph.tiles * n_kv;
    const int runs = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((kWalkWant >> spread) / std::max<int64_t>(1, items), pages / least)));
    set_runs(ph, pages, runs, 1);
    return runs;
}

// Tiles of the prefix beside walks of the own keys: the splits that take least by what was measured of the mixed
// launch (f16). A tile's pair of blocks 3 us, plus 0.4 of the time that the own keys' walks keep the memory busy beside
// it; four pages of a walk (one a wave) 1.25 us and 4 us before them; a slot of every (token, head) 1040 bytes written
// and read at 2.7 TB/s. The own keys are taken to be half of the longest sequence's on average, at 5.5 TB/s, where the
// caller names a longest, and none otherwise. 64 sequences on 8000 shared tokens, 32 heads, own keys up to 1500: 7, 9
// and 13 splits 54.9, 54.5 and 60.4 us, 3 splits 86.5 us; 105 sequences on 3529 tokens, 12 heads, own keys up to 224:
// 3, 4 and 6 splits 43.4, 34.2 and 28.6 us.
constexpr int kTileUnit = 2 * kBlockPages;  // pages
constexpr int kMostRuns = 64;
constexpr double kTilePairUs = 3.0, kTileBeside = 0.4, kWalkStepUs = 1.25, kWalkStartUs = 4.0;
constexpr double kSlotBytesPerUs = 2.7e6, kOwnBytesPerUs = 5.5e6;

void cut_mixed(Launch &l, const EmberRaggedBatch &b, int prefix_pages, int own_pages, bool own_known, int spread) {
    const int64_t tiles = static_cast<int64_t>(l.first.units) * l.first.tiles * b.n_kv;
    const int64_t walks = static_cast<int64_t>(l.second.units) * l.second.tiles * b.n_kv;
    const double slot_us = static_cast<double>(b.T) * b.n_heads * (2 * (kHeadDim + 2) * sizeof(float)) / kSlotBytesPerUs;
    const double page_bytes = 2.0 * kPage * kHeadDim * sizeof(uint16_t);
    const double own_us = own_known ? 0.5 * walks * own_pages * page_bytes / kOwnBytesPerUs : 0.0;
    // Work-groups: tiles one a CU, walks two.
    const int most_tiles = static_cast<int>(std::clamp<int64_t>((kCus >> spread) / tiles, 1, std::min(kMostRuns, (prefix_pages + kTileUnit - 1) / kTileUnit)));
    const int most_walks = static_cast<int>(std::clamp<int64_t>((2 * kCus >> spread) / walks, 1, std::min(kMostRuns, (own_pages + kTileWaves - 1) / kTileWaves)));
    auto least = [&](int most, auto us) {
        int best = 1;
        double best_us = us(1);
        for (int n = 2; n <= most; n++)
            if (const double x = us(n); x < best_us) best = n, best_us = x;
        return best;
    };
    auto steps = [](int pages, int runs, int unit) { return (pages + runs * unit - 1) / (runs * unit); };
    auto walk_us = [&](int n) { return std::max(own_us, kWalkStartUs + kWalkStepUs * steps(own_pages, n, kTileWaves)); };
    const int own_runs = least(most_walks, [&](int n) { return walk_us(n) + n * slot_us; });
    const double beside_us = kWalkStartUs + walk_us(own_runs);
    const int runs = least(most_tiles, [&](int n) {
        return std::max(beside_us, kTilePairUs * steps(prefix_pages, n, kTileUnit) + kTileBeside * own_us) + n * slot_us;
    });
    set_runs(l.first, prefix_pages, runs, kTileUnit);
    set_runs(l.second, own_pages, own_runs, 1);
    l.most_slots = most_tiles + most_walks;
}

Launch plan_prefix(const EmberPrefixAttnArgs &a, int spread) {
    const EmberRaggedBatch &b = a.batch;
    const int G = b.n_heads / b.n_kv;
    const int64_t in_group = std::min(a.max_group, b.T), in_seq = std::min(b.max_query, b.T);
    auto pages_of = [&](int keys) { return std::min(b.max_blocks, keys / kPage + 2); };
    Launch l;
    l.tokens = b.T;
    l.tiled = a.n_groups > 0 && b.dtype == EMBER_DTYPE_F16 && in_group * G > kWalkRows;
    l.most_slots = 0;
    if (a.n_groups > 0) l.first = rows_phase(kPrefixRows, a.n_groups, in_group, G, b.n_kv, l.tiled, 0);
    l.second = rows_phase(kOwnRows, b.S, in_seq, G, b.n_kv, false, 0);
    if (l.tiled) {
        cut_mixed(l, b, pages_of(a.max_prefix), pages_of(a.max_own), a.max_own / kPage < b.max_blocks, spread);
    } else {
        const int fine = b.dtype == EMBER_DTYPE_F16 ? kWalkFine : kWalkFine / 2;  // f32 pages are twice the bytes and the time
        if (a.n_groups > 0) l.most_slots = cut_phase(l.first, b.n_kv, pages_of(a.max_prefix), fine, spread);
        l.most_slots += cut_phase(l.second, b.n_kv, pages_of(a.max_own), fine, spread);
    }
    l.second.slot0 = l.first.splits;
    l.slots = l.first.splits + l.second.splits;
    return l;
}

SpanParams params_of(const EmberRaggedBatch &b, const Launch &l) {
    SpanParams p{};
    p.q = b.q, p.k = b.k_cache, p.v = b.v_cache, p.out = b.out;
    p.query_start = b.query_start, p.positions = b.positions, p.tables = b.block_tables;
    p.q_stride = b.q_stride;
    p.T = b.T, p.S = b.S, p.max_blocks = b.max_blocks, p.n_heads = b.n_heads, p.n_kv = b.n_kv;
    p.G = b.n_heads / b.n_kv, p.num_blocks = b.num_blocks, p.slots = l.slots, p.part_tokens = l.tokens;
    if (l.slots > 1) {
        p.part_acc = static_cast<float *>(b.workspace);
        p.part_ml = p.part_acc + static_cast<int64_t>(l.tokens) * b.n_heads * l.slots * kHeadDim;
    }
    p.window = kNoWindow;
    p.scale_log2 = b.scale * kLog2e;
    return p;
}

template <typename T, int W>
void launch_walk(const SpanParams &p, const Launch &l, unsigned first, unsigned second, hipStream_t stream) {
    hipLaunchKernelGGL((span_walk_kernel<T, W>), dim3(first + second), dim3(W * kWave), 0, stream, p, l.first,
                       l.second, static_cast<int>(first));
}

template <typename T>
hipError_t run(const SpanParams &p, const Launch &l, hipStream_t stream) {
    const unsigned first = static_cast<unsigned>(groups_of(l.first, p.n_kv)), second = static_cast<unsigned>(groups_of(l.second, p.n_kv));
    bool done = first + second == 0;
    if constexpr (sizeof(T) == 2) {
        if (l.tiled && second)
            hipLaunchKernelGGL(span_mixed_kernel, dim3(first + second), dim3(kTileThreads), 0, stream, p, l.first, l.second,
                               static_cast<int>(first));
        else if (l.tiled && first <= kCus)
            hipLaunchKernelGGL(span_tile_kernel<2>, dim3(first), dim3(2 * kTileThreads), 0, stream, p, l.first);
        else if (l.tiled)
            hipLaunchKernelGGL(span_tile_kernel<1>, dim3(first), dim3(kTileThreads), 0, stream, p, l.first);
        else if (!second && first <= kCus)  // a window's work-groups are as wide as their share of the chip
            launch_walk<T, 16>(p, l, first, second, stream);
        done = done || l.tiled || (!second && first <= kCus);
    }
    if (!done && !second && first <= 2 * kCus) launch_walk<T, 8>(p, l, first, second, stream);
    else if (!done) launch_walk<T, 4>(p, l, first, second, stream);
    if (l.slots > 1) {
        constexpr int64_t most = int64_t{1} << 25;  // rows of one launch
        static_assert(most % kMergeWaves == 0 && most * kWave <= UINT32_MAX);
        const int64_t rows = static_cast<int64_t>(p.part_tokens) * p.n_heads;
        for (int64_t first_row = 0; first_row < rows; first_row += most)
            hipLaunchKernelGGL(span_merge_kernel<T>, dim3(static_cast<unsigned>((std::min(most, rows - first_row) + kMergeWaves - 1) / kMergeWaves)),
                               dim3(kMergeWaves * kWave), 0, stream, p, first_row);
    }
    return hipGetLastError();
}

// The launch that the workspace has room for.
template <typename Plan>
int fit(const char *who, const EmberRaggedBatch &b, Plan plan, Launch &l) {
    const int64_t room = b.workspace ? b.workspace_bytes : 0;
    for (int spread = 0; spread <= kLeastSpread; spread++) {
        l = plan(spread);
        if (partial_bytes(b, l.tokens, l.slots) <= room) break;
        if (spread == kLeastSpread)
            return set_error(EMBER_ERR_INVALID, "%s: needs %lld bytes of workspace at least (got %lld)", who,
                             static_cast<long long>(partial_bytes(b, l.tokens, l.slots)), static_cast<long long>(room));
    }
    if (groups_of(l.first, b.n_kv) + groups_of(l.second, b.n_kv) > kMostLaunch)
        return set_error(EMBER_ERR_INVALID, "%s: too many work-groups for one launch (S %d x n_kv %d)", who, b.S, b.n_kv);
    return EMBER_OK;
}

}  // namespace

// A window's workspace holds the partials of these sizes and of smaller batches, which split more: fewer work-groups than
// CUs, so at most kCus tiles of rows in all (of S x max_query tokens; rows of padding behind them have no partials).
int64_t window_workspace_bytes(const EmberWindowAttnArgs &a) {
    const Launch l = plan_window(a, 0);
    const int64_t slots = std::clamp<int64_t>(kCus / a.batch.n_kv, 1, (l.pages + kTileUnit - 1) / kTileUnit);
    const int64_t rows = slots > 1 ? std::min<int64_t>(static_cast<int64_t>(l.tokens) * a.batch.n_heads * slots, kCus * kTileRows) : 0;
    return std::max(partial_bytes(a.batch, l.tokens, l.most_slots), rows * (kHeadDim + 2) * static_cast<int64_t>(sizeof(float)));
}
int64_t shared_prefix_workspace_bytes(const EmberPrefixAttnArgs &a) {
    return partial_bytes(a.batch, a.batch.T, plan_prefix(a, 0).most_slots);
}

int launch_window_attn(const EmberWindowAttnArgs &a, hipStream_t stream) {
    Launch l;
    if (int e = fit("window_attn", a.batch, [&](int spread) { return plan_window(a, spread); }, l)) return e;
    SpanParams p = params_of(a.batch, l);
    p.window = static_cast<uint32_t>(a.window), p.sinks = a.sinks;
    return hip_status(a.batch.dtype == EMBER_DTYPE_F16 ? run<f16>(p, l, stream) : run<float>(p, l, stream), "window_attn");
}

int launch_shared_prefix_attn(const EmberPrefixAttnArgs &a, hipStream_t stream) {
    Launch l;
    if (int e = fit("shared_prefix_attn", a.batch, [&](int spread) { return plan_prefix(a, spread); }, l)) return e;
    SpanParams p = params_of(a.batch, l);
    p.group_start = a.group_start, p.prefix_len = a.prefix_len, p.n_groups = a.n_groups;
    return hip_status(a.batch.dtype == EMBER_DTYPE_F16 ? run<f16>(p, l, stream) : run<float>(p, l, stream), "shared_prefix_attn");
}

}  // namespace ember::hip
