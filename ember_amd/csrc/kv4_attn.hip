// Causal attention of ragged batches over 4-bit pages (ember_hip_kv4_attn).
//
// A page of a kv head is one piece of 2176 bytes that a wave reads in four
// loads: lane l = 16 g + c takes the 16 bytes at 16 (4 c + g) of the K codes
// (key c, dims 32 g .. + 31: one group, one scale byte) and those at 16 l of
// the V codes (keys 4 g .. + 3, dims 8 c .. + 7, a word a key, with the word of
// their four scales). Both are the products' A operands after conversion:
//   S^T = K Q^T    v_mfma_f32_16x16x32_f16, step s over the lane's dims 8 s .. + 7
//                  (the order in which dims are summed is free); row c of q is
//                  column c, so lane l ends with keys 4 g .. + 3 of row c;
//   O^T += V^T P^T the same instruction over the keys of two pages, the
//                  weights where the scores were; tile t holds dims 8 c + t,
//                  two v_perm a page pair up two keys' halves.
// Softmax online in base 2, in f32; weights are f16 and summed as rounded.
//
// Two forms. Few rows (KEYS): the waves of a work-group share the rows and
// take turns at the pages, and meet in LDS. Many rows: each wave has rows of
// its own. A long context is cut into runs of pages for several work-groups;
// the last of them to finish joins the partials, in run order.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "capi_errors.hpp"
#include "four_bit.hpp"
#include "kernels.hpp"

namespace ember::hip {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kStepPages = 4;  // pages that a wave takes at a time
constexpr int kMostRuns = 64;  // runs of pages of one row tile
constexpr int kCounters = 4096;
constexpr int kRowPitch = kHeadDim + 4;  // floats of a row's partial in LDS

struct Kv4Params {
    const f16 *q;
    const uint8_t *pool;
    f16 *out;
    const int32_t *query_start, *positions, *tables;
    float *part_acc, *part_ml;  // [item, run, row of the work-group][128], [...][2]; an item is a row tile of a kv head
    uint32_t *counters;         // [item]
    int64_t q_stride;
    int T, S, max_blocks, n_heads, n_kv, G, num_blocks;
    int tiles, runs, run_pages;
    float scale_log2;
};

// Partials are written and read with device-scope relaxed accesses, which are coherent across the XCDs' L2s; a
// work-group waits for its stores before it counts itself, so what is counted is visible to the last to count.
__device__ __forceinline__ void put2(float *p, float x, float y) {
    const uint64_t v = __float_as_uint(x) | static_cast<uint64_t>(__float_as_uint(y)) << 32;
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float *p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}

__device__ __forceinline__ int clamped(int x, int most) { return min(max(x, 0), most); }

// Eight consecutive dims of a finished row.
__device__ __forceinline__ void store_piece(f16 *dst, const float (&x)[8], float l) {
    f16x8 v;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = static_cast<f16>(filled(l) ? x[i] / l : 0.0f);
    *reinterpret_cast<f16x8 *>(dst) = v;
}

template <int RT, bool KEYS>  // RT tiles of 16 rows a wave
__global__ void __launch_bounds__(kThreads) kv4_attn_kernel(Kv4Params p) {
    constexpr int D = kHeadDim;
    constexpr int kRows = 16 * RT * (KEYS ? 1 : kWaves);  // rows of a work-group
    constexpr int kLdsFloats = KEYS ? kWaves * 16 * RT * (kRowPitch + 2) : 2 * kRows;
    __shared__ float lds[kLdsFloats];
    __shared__ bool last;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int g = lane >> 4, c = lane & 15;
    int rest = static_cast<int>(blockIdx.x);
    const int kvh = rest % p.n_kv;
    rest /= p.n_kv;
    const int tile0 = rest % p.tiles;
    rest /= p.tiles;
    const int run = rest % p.runs, seq = rest / p.runs;
    const int64_t item = (static_cast<int64_t>(seq) * p.tiles + tile0) * p.n_kv + kvh;

    const int t0 = clamped(uniform_load(p.query_start + seq), p.T);
    const int t1 = min(max(uniform_load(p.query_start + seq + 1), t0), p.T);
    const int rows = (t1 - t0) * p.G;
    // More rows than the launch was shaped for: the first run's work-groups take all of them, uncut.
    const bool cut = p.runs > 1 && rows <= p.tiles * kRows;
    if (!cut && run > 0) return;
    const int32_t *const table = p.tables + static_cast<int64_t>(seq) * p.max_blocks;
    const int table_top = p.max_blocks * kPage - 1;

    for (int row0 = tile0 * kRows; row0 < rows; row0 += p.tiles * kRows) {
        const int nrows = min(kRows, rows - row0);
        const int wave_row = KEYS ? 0 : wave * 16 * RT;
        // Positions count up, so a wave's first and last rows bound them.
        auto pos_of = [&](int r) { return p.positions[t0 + (row0 + min(r, nrows - 1)) / p.G]; };
        auto top_of = [&](int r) { return min(max(pos_of(r), -1), table_top); };
        int my_top[RT];
        u32x4 qf[RT][4];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const int row = min(wave_row + 16 * r + c, nrows - 1);
            my_top[r] = top_of(row);
            const f16 *const qp = p.q + (t0 + (row0 + row) / p.G) * p.q_stride + (kvh * p.G + (row0 + row) % p.G) * D + 32 * g;
#pragma unroll
            for (int s = 0; s < 4; s++) qf[r][s] = *reinterpret_cast<const u32x4 *>(qp + 8 * s);
        }
        const int min_top = uniform(top_of(wave_row)), max_top = uniform(top_of(wave_row + 16 * RT - 1));
        const int group_pages = (uniform(top_of(kRows - 1)) + kPage) / kPage;  // of the work-group
        const int active = cut ? max(1, (group_pages + p.run_pages - 1) / p.run_pages) : 1;
        if (run >= active) return;
        const int pages = (max_top + kPage) / kPage;
        const int v0 = cut ? run * p.run_pages : 0, v1 = cut ? min(v0 + p.run_pages, pages) : pages;

        float m[RT], l[RT];
        f32x4 o[RT][8];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            m[r] = kNoKeys, l[r] = 0.0f;
#pragma unroll
            for (int t = 0; t < 8; t++) o[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        constexpr int kStride = KEYS ? kWaves : 1;
        constexpr int kAhead = kWave / kStepPages;  // steps whose block ids a register holds
        const int steps = max(0, v1 - v0 + kStepPages - 1) / kStepPages;
        for (int step0 = KEYS ? wave : 0; step0 < steps; step0 += kStride * kAhead) {
            const int my_page = v0 + (step0 + lane / kStepPages * kStride) * kStepPages + lane % kStepPages;
            const int ids = my_page < v1 ? table[my_page] : -1;
            const int n = min(kAhead, (steps - step0 + kStride - 1) / kStride);
            for (int j = 0; j < n; j++) {
                const int page0 = v0 + (step0 + j * kStride) * kStepPages;
                u32x4 kc[kStepPages], vc[kStepPages];
                uint32_t ks[kStepPages], vs[kStepPages];
#pragma unroll
                for (int i = 0; i < kStepPages; i++) {
                    const int block = __builtin_amdgcn_readlane(ids, j * kStepPages + i);
                    const bool ok = block >= 0 && block < p.num_blocks;  // else no records: the loads give zeros
                    const uint8_t *const base = p.pool + (static_cast<int64_t>(ok ? block : 0) * p.n_kv + kvh) * kKv4Page;
                    const auto d = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, ok ? kKv4Page : 0, kDescWord3);
                    kc[i] = load_desc(d, 64 * c + 16 * g);
                    ks[i] = __builtin_amdgcn_raw_buffer_load_b8(d, kKv4KeyScales + 4 * c + g, 0, kNonTemporal);
                    vc[i] = load_desc(d, kKv4Values + 16 * lane);
                    vs[i] = __builtin_amdgcn_raw_buffer_load_b32(d, kKv4ValueScales + kPage * (c / 4) + 4 * g, 0, kNonTemporal);
                }
                f32x4 s[RT][kStepPages];
#pragma unroll
                for (int i = 0; i < kStepPages; i++) {
#pragma unroll
                    for (int r = 0; r < RT; r++) s[r][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const f16x8 kf = as_f16x8(mx_decode8(kc[i][w], mx_scale(ks[i])));
#pragma unroll
                        for (int r = 0; r < RT; r++) s[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, as_f16x8(qf[r][w]), s[r][i], 0, 0, 0);
                    }
                }
                const int key0 = page0 * kPage;
                if (key0 + kStepPages * kPage - 1 > min_top) {  // some row does not see all of these keys
#pragma unroll
                    for (int i = 0; i < kStepPages; i++)
#pragma unroll
                        for (int v = 0; v < 4; v++) {
                            const int key = key0 + i * kPage + 4 * g + v;
#pragma unroll
                            for (int r = 0; r < RT; r++) s[r][i][v] = key <= my_top[r] ? s[r][i][v] : -INFINITY;
                            // Keys that no row sees may hold anything: their scales are taken as 2^-127, their values so as 0.
                            if (key > max_top) vs[i] &= ~(0xffu << (8 * v));
                        }
                }
                f16x8 wh[RT][kStepPages / 2];
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    float top = s[r][0][0];
#pragma unroll
                    for (int i = 0; i < kStepPages; i++)
#pragma unroll
                        for (int v = 0; v < 4; v++) top = fmaxf(top, s[r][i][v]);
                    top = groups_max(top) * p.scale_log2;
                    const float mn = fmaxf(m[r], below(top, kMostExponent));
                    const float corr = exp2_hw(m[r] - mn);
                    m[r] = mn;
                    float mul = p.scale_log2, add = -mn;
                    if (const bool far = fabsf(mn) >= kFar; __builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
                        for (int i = 0; i < kStepPages; i++)
#pragma unroll
                            for (int v = 0; v < 4; v++) s[r][i][v] = far ? s[r][i][v] * mul + add : __builtin_fmaf(s[r][i][v], mul, add);
                        mul = 1.0f, add = 0.0f;
                    }
                    l[r] = l[r] * corr;
                    const f16x2 ones = {static_cast<f16>(1.0f), static_cast<f16>(1.0f)};
#pragma unroll
                    for (int i = 0; i < kStepPages; i++) {
#pragma unroll
                        for (int v = 0; v < 4; v++) wh[r][i / 2][i % 2 * 4 + v] = static_cast<f16>(exp2_hw(__builtin_fmaf(s[r][i][v], mul, add)));
#pragma unroll
                        for (int v = 0; v < 4; v += 2)
                            l[r] = __builtin_amdgcn_fdot2(f16x2{wh[r][i / 2][i % 2 * 4 + v], wh[r][i / 2][i % 2 * 4 + v + 1]}, ones, l[r], false);
                    }
#pragma unroll
                    for (int t = 0; t < 8; t++) o[r][t] = o[r][t] * corr;
                }
#pragma unroll
                for (int i = 0; i < kStepPages; i += 2) {
                    u32x4 val[2][4];  // [page][key % 4]: dims 8 c .. + 7
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int v = 0; v < 4; v++) val[h][v] = mx_decode8(vc[i + h][v], mx_scale(vs[i + h], v));
                    auto tile = [&](auto index) {
                        constexpr int t = decltype(index)::value;
                        const f16x4 a = value_tile<t>(val[0]), b = value_tile<t>(val[1]);
                        const f16x8 vt = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                        for (int r = 0; r < RT; r++) o[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, wh[r][i / 2], o[r][t], 0, 0, 0);
                    };
                    tile(std::integral_constant<int, 0>{}), tile(std::integral_constant<int, 1>{});
                    tile(std::integral_constant<int, 2>{}), tile(std::integral_constant<int, 3>{});
                    tile(std::integral_constant<int, 4>{}), tile(std::integral_constant<int, 5>{});
                    tile(std::integral_constant<int, 6>{}), tile(std::integral_constant<int, 7>{});
                }
            }
        }
#pragma unroll
        for (int r = 0; r < RT; r++) l[r] = groups_sum(l[r]);

        // The row's place in out.
        auto at_of = [&](int row) {
            return static_cast<int64_t>(t0 + (row0 + row) / p.G) * p.n_heads + kvh * p.G + (row0 + row) % p.G;
        };
        auto emit = [&](int row, int dim, const float (&x)[8], float row_m, float row_l) {
            if (active == 1) return store_piece(p.out + at_of(row) * D + dim, x, row_l);
            const int64_t slot = (item * p.runs + run) * kRows + row;
#pragma unroll
            for (int i = 0; i < 8; i += 2) put2(p.part_acc + slot * D + dim + i, x[i], x[i + 1]);
            if (dim == 0) put2(p.part_ml + slot * 2, row_m, row_l);
        };
        if constexpr (KEYS) {
            float *const red_m = lds + kWaves * kRows * kRowPitch, *const red_l = red_m + kWaves * kRows;
            __syncthreads();  // of the rows before these
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const int row = 16 * r + c;
                float *const dst = lds + (wave * kRows + row) * kRowPitch + 32 * g;
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    *reinterpret_cast<f32x4 *>(dst + 8 * v) = f32x4{o[r][0][v], o[r][1][v], o[r][2][v], o[r][3][v]};
                    *reinterpret_cast<f32x4 *>(dst + 8 * v + 4) = f32x4{o[r][4][v], o[r][5][v], o[r][6][v], o[r][7][v]};
                }
                if (g == 0) red_m[wave * kRows + row] = m[r], red_l[wave * kRows + row] = l[r];
            }
            __syncthreads();
            for (int i = tid; i < nrows * 16; i += kThreads) {
                const int row = i / 16, dim = i % 16 * 8;
                float M = kNoKeys, L = 0.0f, x[8] = {};
#pragma unroll
                for (int w = 0; w < kWaves; w++) M = fmaxf(M, red_m[w * kRows + row]);
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const float part = red_l[w * kRows + row], f = filled(part) ? exp2_hw(red_m[w * kRows + row] - M) : 0.0f;
                    L = L + part * f;
                    const float *const src = lds + (w * kRows + row) * kRowPitch + dim;
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = x[e] + src[e] * f;
                }
                emit(row, dim, x, M, L);
            }
        } else {
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const int row = wave_row + 16 * r + c;
                if (row < nrows)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const float x[8] = {o[r][0][v], o[r][1][v], o[r][2][v], o[r][3][v], o[r][4][v], o[r][5][v], o[r][6][v], o[r][7][v]};
                        emit(row, 32 * g + 8 * v, x, m[r], l[r]);
                    }
            }
        }
        if (active == 1) continue;

        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0) {
            uint32_t *const counter = p.counters + item;
            last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == static_cast<uint32_t>(active);
            if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last) return;
        for (int i = tid; i < nrows * 16; i += kThreads) {
            const int row = i / 16, dim = i % 16 * 8;
            const int64_t slot0 = item * p.runs * kRows + row;  // and one every kRows
            float M = kNoKeys, L = 0.0f, x[8] = {};
            for (int s = 0; s < active; s++) M = fmaxf(M, get2(p.part_ml + (slot0 + s * kRows) * 2).x);
            for (int s = 0; s < active; s++) {
                const float2 ml = get2(p.part_ml + (slot0 + s * kRows) * 2);
                const float f = filled(ml.y) ? exp2_hw(ml.x - M) : 0.0f;
                L = L + ml.y * f;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float2 a = get2(p.part_acc + (slot0 + s * kRows) * D + dim + e);
                    x[e] = x[e] + a.x * f, x[e + 1] = x[e + 1] + a.y * f;
                }
            }
            store_piece(p.out + at_of(row) * D + dim, x, L);
        }
        return;  // a cut step has one tile a work-group
    }
}

// ---- host ----

constexpr int64_t kMostGroups = 1 << 20;                   // row tiles of a launch beyond which work-groups take several
constexpr int64_t kMostLaunch = UINT32_MAX / kThreads;     // HIP's bound on a launch's threads
constexpr int kWant = 1024;                                // work-groups that fill the chip

struct Plan {
    int rows = 16;  // of a work-group
    int tiles = 1, runs = 1, run_pages = 1;
    int most_runs = 1;  // for any number of sequences
};

constexpr int kForms[] = {16, 32, 128};  // rows of a work-group

int64_t partial_bytes(int64_t groups, int rows) { return kCounters * 4 + groups * rows * (kHeadDim + 2) * 4; }

// The plan for at most `most` rows of a sequence and a kv head.
Plan plan(const EmberKv4AttnArgs &a, int64_t most, int64_t room) {
    const EmberRaggedBatch &b = a.batch;
    Plan l;
    l.rows = most <= 16 ? 16 : most <= 32 ? 32 : 128;
    const int64_t units = static_cast<int64_t>(b.S) * b.n_kv;
    l.tiles = static_cast<int>(std::clamp<int64_t>((most + l.rows - 1) / l.rows, 1, std::max<int64_t>(1, kMostGroups / units)));
    const int pages = std::min(b.max_blocks, a.max_context / kPage + 1);
    const int64_t items = units * l.tiles;
    l.most_runs = std::clamp(pages / (kStepPages * 4), 1, kMostRuns);
    int64_t runs = items > kCounters ? 1 : std::clamp<int64_t>(kWant / items, 1, l.most_runs);
    while (runs > 1 && partial_bytes(items * runs, l.rows) > room) runs--;
    l.run_pages = static_cast<int>((pages + runs * kStepPages - 1) / (runs * kStepPages)) * kStepPages;  // a step is of one run
    l.runs = (pages + l.run_pages - 1) / l.run_pages;
    return l;
}

int64_t most_rows(const EmberRaggedBatch &b) { return static_cast<int64_t>(std::min(b.max_query, b.T)) * (b.n_heads / b.n_kv); }

}  // namespace

// Cut launches have at most kWant work-groups, and as many as the sequences' items and runs give: the largest of what each
// form up to this one could use.
int64_t kv4_workspace_bytes(const EmberKv4AttnArgs &a) {
    const int64_t most = most_rows(a.batch);
    int64_t bytes = 0;
    for (int rows : kForms) {
        const Plan l = plan(a, std::min<int64_t>(most, rows == 128 ? most : rows), 0);
        const int64_t groups = std::min<int64_t>(kWant, static_cast<int64_t>(a.batch.S) * a.batch.n_kv * l.tiles * l.most_runs);
        if (l.most_runs > 1 && a.batch.n_kv * 2 <= kWant) bytes = std::max(bytes, partial_bytes(groups, l.rows));
    }
    return bytes;
}

int launch_kv4_attn(const EmberKv4AttnArgs &a, hipStream_t stream) {
    const EmberRaggedBatch &b = a.batch;
    const Plan l = plan(a, most_rows(b), b.workspace ? b.workspace_bytes : 0);
    const int64_t groups = static_cast<int64_t>(b.S) * b.n_kv * l.tiles * l.runs;
    if (groups > kMostLaunch)
        return set_error(EMBER_ERR_INVALID, "kv4_attn: too many work-groups for one launch (S %d x n_kv %d)", b.S, b.n_kv);
    Kv4Params p{};
    p.q = static_cast<const f16 *>(b.q), p.pool = static_cast<const uint8_t *>(b.k_cache), p.out = static_cast<f16 *>(b.out);
    p.query_start = b.query_start, p.positions = b.positions, p.tables = b.block_tables;
    p.q_stride = b.q_stride;
    p.T = b.T, p.S = b.S, p.max_blocks = b.max_blocks, p.n_heads = b.n_heads, p.n_kv = b.n_kv, p.G = b.n_heads / b.n_kv;
    p.num_blocks = b.num_blocks;
    p.tiles = l.tiles, p.runs = l.runs, p.run_pages = l.run_pages;
    if (l.runs > 1) {
        p.counters = static_cast<uint32_t *>(b.workspace);
        p.part_acc = reinterpret_cast<float *>(p.counters + kCounters);
        p.part_ml = p.part_acc + groups * l.rows * kHeadDim;
    }
    p.scale_log2 = b.scale * kLog2e;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream, p); };
    if (l.rows == 16) go(kv4_attn_kernel<1, true>);
    else if (l.rows == 32) go(kv4_attn_kernel<2, true>);
    else go(kv4_attn_kernel<2, false>);
    return hip_status(hipGetLastError(), "kv4_attn");
}

}  // namespace ember::hip
