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
// Softmax online in base 2: maxima and sums in f32; a weight is f16 and enters
// the sum as rounded, so that sum and products see the same weights. A row's
// reference is not its maximum but 7 below it, and moves only when a score
// exceeds it by 15, short of f16's end: a weight keeps its 11 bits down to
// 2^-21 of the largest, and the accumulators are seldom rescaled. f16 because
// the matrix unit takes both operands in one type at this rate; it costs 2.9e-4
// against float64 in place of the 2.1e-4 of the outputs' rounding alone.
//
// Two forms. Up to 32 rows of a kv head and sequence (decode, speculative
// runs): the walk, whose four waves take turns at the pages and convert them in
// registers. More (prompts): the tile, 128 rows on blocks of keys converted
// once into LDS. In both, either a work-group has an item (a row tile of a
// sequence), or the work-groups of a kv head share the keys of all items out
// evenly; then the last to finish of an item joins its partials, in the order
// of the keys: the bits do not depend on who that is.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "capi_errors.hpp"
#include "four_bit.hpp"
#include "kernels.hpp"

namespace ember::hip {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kLeastUnits = 8;  // of a work-group's share
constexpr int kRowPitch = kHeadDim + 4;  // floats of a row's partial in LDS

constexpr int kMostDealt = 256;  // sequences of a launch whose items are dealt by length

struct Kv4Params {
    const f16 *q;
    const uint8_t *pool;
    f16 *out;
    const int32_t *query_start, *positions, *tables;
    float *part_acc, *part_ml;  // [work-group, slot][row][128], [...][2]
    uint32_t *counters;         // [work-group]
    int64_t q_stride;
    int T, S, max_blocks, n_heads, n_kv, G, num_blocks;
    int workers;  // work-groups of a kv head
    int tiles;    // entries of a sequence: its row tiles, those past the hint together in the last
    int least, most;  // rows of the sequences that this launch is for
    int shift;    // a unit of their shares is 2^shift steps of pages
    int round;    // without sharing: sequences whose items fill the CUs once, if they are dealt by length, else 0
    float scale_log2;
};

// Partials are written and read at device scope (sc1), which the XCDs' L2s do not keep from one another; a work-group
// waits for its stores before it counts itself, so what is counted is visible to the last to count.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
constexpr int kDeviceScope = 16;  // cache-policy bit sc1 of a gfx950 buffer access

__device__ __forceinline__ __amdgpu_buffer_rsrc_t partials(const float *base, int64_t at, int floats) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(base) + at, 0, floats * static_cast<int>(sizeof(float)), kDescWord3);
}

__device__ __forceinline__ int clamped(int x, int most) { return min(max(x, 0), most); }

// Eight consecutive dims of a finished row.
__device__ __forceinline__ void store_piece(f16 *dst, const float (&x)[8], float l) {
    f16x8 v;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = static_cast<f16>(filled(l) ? x[i] / l : 0.0f);
    *reinterpret_cast<f16x8 *>(dst) = v;
}

// The partials of a slot: ROWS rows of 128, and of (max, sum).
template <int ROWS>
struct Partials {
    __amdgpu_buffer_rsrc_t acc, ml;
    __device__ __forceinline__ Partials(const Kv4Params &p, int slot)
        : acc(partials(p.part_acc, static_cast<int64_t>(slot) * ROWS * kHeadDim, ROWS * kHeadDim)),
          ml(partials(p.part_ml, static_cast<int64_t>(slot) * ROWS * 2, ROWS * 2)) {}
    __device__ __forceinline__ void put4(int row, int dim, const f32x4 &x) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), acc, (row * kHeadDim + dim) * static_cast<int>(sizeof(float)), 0, kDeviceScope);
    }
    __device__ __forceinline__ void put_ml(int row, float m, float l) const {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, ml, 8 * row, 0, kDeviceScope);
    }
    __device__ __forceinline__ float2 get_ml(int row) const {
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(ml, 8 * row, 0, kDeviceScope));
        return make_float2(__uint_as_float(v[0]), __uint_as_float(v[1]));
    }
    // A tile's, as its lanes hold them: operand i of a lane is 16 bytes, a wave's side by side.
    static __device__ __forceinline__ int lane_at(int wave, int i, int lane) { return ((wave * 16 + i) * kWave + lane) * 16; }
    __device__ __forceinline__ void put_lane(int wave, int i, int lane, const f32x4 &x) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), acc, lane_at(wave, i, lane), 0, kDeviceScope);
    }
    __device__ __forceinline__ u32x4 get_lane(int wave, int i, int lane) const {
        return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(acc, lane_at(wave, i, lane), 0, kDeviceScope));
    }
    __device__ __forceinline__ u32x4 get4(int row, int dim) const {
        return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(acc, (row * kHeadDim + dim) * static_cast<int>(sizeof(float)), 0, kDeviceScope));
    }
};

__device__ __forceinline__ float row16_max(float x) {
    x = fmaxf(x, dpp_mov<kDppQuadXor1>(x));
    x = fmaxf(x, dpp_mov<kDppQuadXor2>(x));
    x = fmaxf(x, dpp_mov<kDppRowHalfMirror>(x));
    return fmaxf(x, dpp_mov<kDppRowMirror>(x));
}

// Counts this work-group, whose partials are written, and says whether it is the last of n. Leaves the counter at 0.
__device__ __forceinline__ bool last_of(uint32_t *counter, int n, bool &last) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == static_cast<uint32_t>(n);
        if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return last;
}

// Joins n partials of nrows rows, slot_of(0) .. slot_of(n - 1) in that order, kMergePieces at a time. 16 lanes share a
// row, 8 dims each; where the rows leave threads over, groups of them take every groups-th partial, and their sums are
// added in group order.
constexpr int kMergePieces = 32;
constexpr int merge_floats(int rows, int threads) { return 2 * rows * kMergePieces + threads * 8; }

template <int ROWS, int THREADS, typename Slot, typename At>
__device__ __forceinline__ void merge_partials(const Kv4Params &p, int n, int nrows, float *lds, Slot slot_of, At at_of) {
    constexpr int kPitch = kMergePieces;
    float *const top = lds, *const sum = top + ROWS * kPitch, *const x_lds = sum + ROWS * kPitch;  // [row][partial]
    const int tid = static_cast<int>(threadIdx.x), lanes = nrows * 16;
    const int groups = max(1, THREADS / lanes), group = groups > 1 ? tid / lanes : 0;
    for (int i0 = 0; i0 < lanes; i0 += THREADS) {  // (one round where there are groups)
        const int i = i0 + (groups > 1 ? tid % lanes : tid);
        const bool mine = i < lanes && group < groups;
        const int row = min(i / 16, nrows - 1), dim = i % 16 * 8;
        float M = kNoKeys, L = 0.0f, x[8] = {};
        for (int n0 = 0; n0 < n; n0 += kMergePieces) {
            const int some = min(kMergePieces, n - n0);
            __syncthreads();
            for (int k = tid; k < nrows * some; k += THREADS) {
                const float2 ml = Partials<ROWS>(p, slot_of(n0 + k / nrows)).get_ml(k % nrows);
                top[k % nrows * kPitch + k / nrows] = ml.x, sum[k % nrows * kPitch + k / nrows] = ml.y;
            }
            __syncthreads();
            // Lane i % 16 of a row takes every 16th of its weights.
            float now = M;
#pragma unroll
            for (int k = 0; k < kMergePieces; k += 16)
                if (const int at = k + i % 16; at < some) now = fmaxf(now, top[row * kPitch + at]);
            now = row16_max(now);
            const float corr = exp2_hw(M - now);
            M = now;
            L = L * corr;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = x[e] * corr;
            float add = 0.0f, weight[kMergePieces / 16];
#pragma unroll
            for (int k = 0; k < kMergePieces; k += 16) {
                const int at = row * kPitch + min(k + i % 16, some - 1);
                weight[k / 16] = filled(sum[at]) ? exp2_hw(top[at] - M) : 0.0f;
                add = add + (k + i % 16 < some ? sum[at] * weight[k / 16] : 0.0f);
            }
            L = L + row16_sum(add);
            __syncthreads();
            if (mine && group == 0)
#pragma unroll
                for (int k = 0; k < kMergePieces; k += 16) top[row * kPitch + k + i % 16] = weight[k / 16];
            __syncthreads();
            constexpr int kInFlight = 4;
            for (int k0 = group; k0 < some && mine; k0 += groups * kInFlight) {
                u32x4 part[kInFlight][2];
#pragma unroll
                for (int f = 0; f < kInFlight; f++) {
                    const Partials<ROWS> from(p, slot_of(n0 + min(k0 + f * groups, some - 1)));
                    part[f][0] = from.get4(row, dim), part[f][1] = from.get4(row, dim + 4);
                }
#pragma unroll
                for (int f = 0; f < kInFlight; f++) {
                    if (k0 + f * groups >= some) break;
                    const float w = top[row * kPitch + k0 + f * groups];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = x[e] + __uint_as_float(part[f][e / 4][e % 4]) * w;
                }
            }
        }
        if (groups > 1) {
#pragma unroll
            for (int e = 0; e < 8; e++) x_lds[e * THREADS + tid] = x[e];
            __syncthreads();
            if (group == 0)
                for (int k = 1; k < groups; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = x[e] + x_lds[e * THREADS + k * lanes + i];
        }
        if (mine && group == 0) store_piece(p.out + at_of(row) * kHeadDim + dim, x, L);
    }
}

// How U units of work are shared out: worker j of n takes units start(j) .. start(j + 1) - 1, but a start that lies
// within `near` units of an item's border moves to the nearer one: a cut item costs its partials and a merge.
struct Shares {
    int each, more, near;  // `more` of the workers take one unit more than `each`
    __device__ __forceinline__ Shares(int units, int workers)
        : each(units / workers), more(units - each * workers), near(max(1, each / 8)) {}
    __device__ __forceinline__ Shares(int each, int more, int near) : each(each), more(more), near(near) {}
    __device__ __forceinline__ int start(int j) const { return j * each + min(j, more); }
    __device__ __forceinline__ int worker_of(int unit) const {
        const int high = more * (each + 1);
        return unit < high ? unit / (each + 1) : more + (unit - high) / each;
    }
    // A start x within the item of units a .. b - 1.
    __device__ __forceinline__ int moved(int x, int a, int b) const {
        if (x - a <= near && x - a <= b - x) return a;
        return b - x <= near ? b : x;
    }
};

// A part of an item (a row tile of a sequence for a kv head) that a work-group takes: units x .. stop - 1 of the item's
// a .. b - 1, a unit being 2^shift steps of keys.
struct Part {
    int seq, t0, rows, tile;  // the sequence, its first token and its rows; the row tile
    int a, b, x, stop;
    int top;  // the highest key of the tile's rows (of the sequence's, for tiles past the hint)
    __device__ __forceinline__ bool whole() const { return x == a && stop == b; }
};

// The parts of a work-group, in order. With workers, the work-groups of a kv head share the units of all items evenly,
// found by each wave for itself from the sequences' lengths: 64 entries a load, a scan over the lanes. Without, a
// work-group has an entry. An entry is a row tile of a sequence; the sequence's last one is all tiles that are left.
template <int ROWS, int KEYS>  // of a tile, of a step
struct Parts {
    const Kv4Params &p;
    const int lane, worker;
    int workers;
    // Lane i: entry 64 chunk + i. Its sequence's first token and rows, its first tile and number of them, their highest
    // key and units each; units up to it, and before the chunk. The next part begins in lane `at`.
    int seq_t0, seq_rows, first_tile, n_tiles, entry_top, entry_units;
    int upto, before = 0, chunk = 0, at = 0;
    int begin = 0, x = 0, end;
    Shares shares{0, 0, 0};

    struct Raw {
        int start, stop, guess;  // the guess: the last position of a sequence of a pure decode step
    };
    __device__ __forceinline__ int sequence(int e) const { return min(p.tiles == 1 ? e : e / p.tiles, p.S - 1); }
    __device__ __forceinline__ Raw fetch(int e) const {
        const int s = sequence(e);
        return {p.query_start[s], p.query_start[s + 1], p.positions[min(s, p.T - 1)]};
    }
    __device__ __forceinline__ int load(int e) { return settle(e, fetch(e)); }
    __device__ __forceinline__ int settle(int e, const Raw &raw) {
        const int s = sequence(e), k = p.tiles == 1 ? 0 : e - s * p.tiles;
        const int t0 = clamped(raw.start, p.T), t1 = min(max(raw.stop, t0), p.T);
        int pos = raw.guess;
        if (__builtin_amdgcn_ballot_w64(t1 - 1 != s)) pos = p.positions[max(t1 - 1, 0)];
        seq_t0 = t0, seq_rows = (t1 - t0) * p.G;
        const int all = e < p.S * p.tiles && seq_rows >= p.least && seq_rows <= p.most ? (seq_rows + ROWS - 1) / ROWS : 0;
        first_tile = k, n_tiles = k == p.tiles - 1 ? max(all - k, 0) : k < all ? 1 : 0;
        // Positions count up: those behind the tile's last row are known from the sequence's last.
        if (p.tiles > 1 && k < p.tiles - 1) pos = max(pos, -1) - (max(seq_rows - 1, 0) / p.G - (min((k + 1) * ROWS, max(seq_rows, 1)) - 1) / p.G);
        entry_top = min(max(pos, -1), p.max_blocks * kPage - 1);
        const int steps = max(1, (entry_top + KEYS) / KEYS);
        entry_units = (steps + (1 << p.shift) - 1) >> p.shift;
        return n_tiles * entry_units;
    }
    __device__ __forceinline__ int scan(int v) const {  // inclusive, over the lanes
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int y = __shfl_up(v, o, kWave);
            v += lane >= o ? y : 0;
        }
        return v;
    }
    // The entry of a work-group by length: the longest to the first, and the other way round in every second round, so that
    // a CU's first item and its second are together about as long as any other's. The k-th largest, found bit by bit.
    __device__ __forceinline__ void deal() {
        const int turn = worker / p.round, first = turn * p.round;
        int k = turn % 2 ? first + min(p.round, p.S - first) - 1 - (worker - first) : worker;
        const int top = 1 << (31 - __builtin_clz(max(p.max_blocks, 1)));  // of an item; entries of several tiles count as 2 top - 1 at most
        Raw raw[kMostDealt / kWave];
        int units[kMostDealt / kWave];
#pragma unroll
        for (int c = 0; c < kMostDealt / kWave; c++)
            if (c < chunks()) raw[c] = fetch(c * kWave + lane);
#pragma unroll
        for (int c = 0; c < kMostDealt / kWave; c++)
            if (units[c] = -1; c < chunks()) {
                upto = settle(c * kWave + lane, raw[c]);
                units[c] = c * kWave + lane < p.S ? min(upto, 2 * top - 1) : -1;
            }
        auto count = [&](int least) {
            int n = 0;
#pragma unroll
            for (int c = 0; c < kMostDealt / kWave; c++) n += __popcll(__builtin_amdgcn_ballot_w64(units[c] >= least));
            return n;
        };
        int value = 0;
        for (int bit = top; bit > 0; bit >>= 1) value += count(value + bit) > k ? bit : 0;
        k -= count(value + 1);
#pragma unroll
        for (int c = 0; c < kMostDealt / kWave; c++) {
            const uint64_t same = __builtin_amdgcn_ballot_w64(units[c] == value);
            const uint64_t it = __builtin_amdgcn_ballot_w64(units[c] == value && __popcll(same & ((1ull << lane) - 1)) == k);
            if (it) {
                chunk = c, at = __builtin_ctzll(it);
                if (chunks() > 1) upto = settle(c * kWave + lane, raw[c]);
            }
            k -= __popcll(same);
        }
        end = __builtin_amdgcn_readlane(upto, at);
    }
    __device__ __forceinline__ int chunks() const { return (p.S * p.tiles + kWave - 1) / kWave; }

    __device__ __forceinline__ Parts(const Kv4Params &params, int lane, int worker) : p(params), lane(lane), worker(worker), workers(params.workers) {
        if (workers == 0) {
            if (p.round > 0) {
                deal();
                return;
            }
            upto = load(worker);
            end = upto = uniform(upto);
            chunk = worker / kWave, at = worker % kWave;
            return;
        }
        upto = scan(load(lane));
        int units = __builtin_amdgcn_readlane(upto, kWave - 1), chunk_units = units;
        if (chunks() > 1) {  // lane k: the units of chunk k
            for (int k = 1; k < chunks(); k++) {
                const int sum = __builtin_amdgcn_readlane(scan(load(k * kWave + lane)), kWave - 1);
                chunk_units = lane == k ? sum : chunk_units;
            }
            chunk_units = scan(lane < chunks() ? chunk_units : 0);
            units = __builtin_amdgcn_readlane(chunk_units, kWave - 1);
        }
        workers = min(workers, max(1, units / kLeastUnits));
        if (worker >= workers) {
            end = 0;
            return;
        }
        shares = Shares(units, workers);
        x = begin = shares.start(worker), end = shares.start(worker + 1);
        if (chunks() > 1) {  // the chunk of the first unit
            chunk = __popcll(__builtin_amdgcn_ballot_w64(lane < chunks() && chunk_units <= begin));
            before = chunk > 0 ? __builtin_amdgcn_readlane(chunk_units, chunk - 1) : 0;
            upto = scan(load(chunk * kWave + lane));
        }
        at = __popcll(__builtin_amdgcn_ballot_w64(before + upto <= begin));
    }

    __device__ __forceinline__ bool next(Part &part) {
        while (x < end) {
            if (at == kWave) {
                before += __builtin_amdgcn_readlane(upto, kWave - 1);
                if (++chunk >= chunks()) return false;
                upto = scan(load(chunk * kWave + lane));
                at = 0;
            }
            const int entry_end = before + __builtin_amdgcn_readlane(upto, at);
            if (entry_end <= x) {
                at++;
                continue;
            }
            const int entry = chunk * kWave + at;
            part.seq = p.tiles == 1 ? entry : entry / p.tiles;
            part.t0 = __builtin_amdgcn_readlane(seq_t0, at), part.rows = __builtin_amdgcn_readlane(seq_rows, at);
            // The item is the `left`th of its entry's from the end.
            const int units = __builtin_amdgcn_readlane(entry_units, at), tiles = __builtin_amdgcn_readlane(n_tiles, at);
            const int left = tiles == 1 ? 1 : (entry_end - x + units - 1) / units;
            part.tile = __builtin_amdgcn_readlane(first_tile, at) + tiles - left;
            part.b = entry_end - (left - 1) * units, part.a = part.b - units;
            part.top = __builtin_amdgcn_readlane(entry_top, at);
            if (workers > 0 && x == begin) {
                x = shares.moved(x, part.a, part.b);
                if (x == part.b) continue;  // the one before takes it
            }
            part.x = x;
            part.stop = end >= part.b ? part.b : shares.moved(end, part.a, part.b);
            if (part.stop == part.a) return false;
            x = part.stop == part.b ? part.b : end;
            return true;
        }
        return false;
    }

    // The work-groups that have parts of an item that is cut.
    __device__ __forceinline__ void holders(const Part &part, int &from, int &to) const {
        from = shares.worker_of(part.a), to = shares.worker_of(part.b - 1);
        if (from + 1 < workers && shares.start(from + 1) < part.b && shares.moved(shares.start(from + 1), part.a, part.b) == part.a) from++;
        if (to > 0 && shares.start(to) >= part.a && shares.moved(shares.start(to), part.a, part.b) == part.b) to--;
        from = clamped(from, workers - 1), to = clamped(to, workers - 1);  // (an invalid query_start could ask for any)
    }
    // A work-group has two slots for partials: of an item that it begins, and of one that began before it.
    __device__ __forceinline__ int slot(int kvh, int holder, bool begins) const { return 2 * (kvh * p.workers + holder) + (begins ? 1 : 0); }
};

// Up to 16 RT rows a work-group, W waves that take turns at steps of P pages.
//
// Bound by what a CU takes in, 27 to 43 GB/s however many waves ask: so the
// pages of a wave's next step are on their way during a whole step, and where
// contexts are long all CUs have the same share. With few keys, by a launch's
// chain of trips to memory (lengths, page ids, pages, out).
// Measured, 8 kv heads: 1 sequence of 640 keys 7.4 us, of 131,000 32 (4.4
// TB/s); 32 of 256 to 4095 20.7 (4.3 TB/s); 8 of 30,000 to 131,000 135 (6.1
// TB/s); 64 of 512 to 4096 with up to 5 tokens each 30.6 (5.3 TB/s).
template <int RT, int W, int P>
__global__ void __launch_bounds__(W *kWave, 2) kv4_walk_kernel(Kv4Params p) {
    constexpr int D = kHeadDim, kRows = 16 * RT, kThreads = W * kWave;
    constexpr int kLdsFloats = W * kRows * (kRowPitch + 2);
    static_assert(merge_floats(kRows, kThreads) <= kLdsFloats);
    __shared__ __align__(16) float lds[kLdsFloats];
    __shared__ bool last;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int g = lane >> 4, c = lane & 15;
    const int kvh = static_cast<int>(blockIdx.x) % p.n_kv, worker = static_cast<int>(blockIdx.x) / p.n_kv;
    const int table_top = p.max_blocks * kPage - 1;
    const uint8_t *const pool = p.pool + kvh * kKv4Page;
    const uint32_t block_bytes = static_cast<uint32_t>(p.n_kv) * kKv4Page;

    __builtin_amdgcn_s_setprio(3);  // up to the first pages, which the CU's other waves would delay
    Parts<kRows, P * kPage> parts(p, lane, worker);
    Part part;
    while (parts.next(part)) {
        const int t0 = part.t0, rows = part.rows;
        const int row0 = part.tile * kRows, nrows = min(kRows, rows - row0);
        const int32_t *const table = p.tables + static_cast<int64_t>(part.seq) * p.max_blocks;
        // Step i of this wave: pages (wave + i W) P .. of the part; lane P i + j holds the id of its page j.
        constexpr int kAhead = kWave / P;
        const int v0 = ((part.x - part.a) << p.shift) * P;
        const int lane_page = (wave + lane / P * W) * P + lane % P;
        auto id_at = [&](int page) { return page < p.max_blocks ? table[page] : -1; };
        const int first_ids = id_at(v0 + lane_page);
        // Positions count up, so the first and last rows bound them.
        auto top_of = [&](int row) { return min(max(p.positions[t0 + (row0 + row) / p.G], -1), table_top); };
        const bool one_token = rows == p.G;
        int my_top[RT];
        u32x4 qf[RT][4];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const int row = min(16 * r + c, nrows - 1);
            const f16 *const qp = p.q + (t0 + (row0 + row) / p.G) * p.q_stride + (kvh * p.G + (row0 + row) % p.G) * D + 32 * g;
#pragma unroll
            for (int s = 0; s < 4; s++) qf[r][s] = *reinterpret_cast<const u32x4 *>(qp + 8 * s);
        }
        int min_top = part.top, max_top = part.top;
        if (one_token) {
#pragma unroll
            for (int r = 0; r < RT; r++) my_top[r] = max_top;
        } else {
#pragma unroll
            for (int r = 0; r < RT; r++) my_top[r] = top_of(min(16 * r + c, nrows - 1));
            min_top = uniform(top_of(0)), max_top = uniform(top_of(nrows - 1));
        }
        const int pages = (max_top + kPage) / kPage;
        const int v1 = part.stop == part.b ? pages : min(((part.stop - part.a) << p.shift) * P, pages);

        float m[RT], l[RT];
        f32x4 o[RT][8];  // o[t][v]: dim 32 g + 8 v + t of column c
#pragma unroll
        for (int r = 0; r < RT; r++) {
            m[r] = kNoKeys, l[r] = 0.0f;
#pragma unroll
            for (int t = 0; t < 8; t++) o[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const int steps = max(0, v1 - v0 + P - 1) / P;
        for (int step0 = wave; step0 < steps; step0 += W * kAhead) {
            const int page_base = v0 + (step0 - wave) * P;
            const int my_page = page_base + lane_page;
            int ids = step0 == wave ? first_ids : id_at(my_page);
            ids = my_page < v1 ? ids : -1;
            const int n = min(kAhead, (steps - step0 + W - 1) / W);
            struct Step {
                u32x4 kc[P], vc[P];
                uint32_t ks[P], vs[P];
            };
            // A page that is not there, or past the part's last, has no records: its loads give zeros.
            auto fetch = [&](Step &to, int j) {
#pragma unroll
                for (int i = 0; i < P; i++) {
                    const uint32_t block = j < kAhead ? __builtin_amdgcn_readlane(ids, (j * P + i) % kWave) : ~0u;
                    const bool ok = block < static_cast<uint32_t>(p.num_blocks);
                    const auto d = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(pool) + static_cast<uint64_t>(ok ? block : 0) * block_bytes, 0,
                                                                     ok ? kKv4Page : 0, kDescWord3);
                    to.kc[i] = load_desc(d, 64 * c + 16 * g);
                    to.ks[i] = __builtin_amdgcn_raw_buffer_load_b8(d, kKv4KeyScales + 4 * c + g, 0, kNonTemporal);
                    to.vc[i] = load_desc(d, kKv4Values + 16 * lane);
                    to.vs[i] = __builtin_amdgcn_raw_buffer_load_b32(d, kKv4ValueScales + kPage * (c / 4) + 4 * g, 0, kNonTemporal);
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            // Step j, with the next one's pages on their way.
            auto consume = [&](Step &at, Step &next, int j) {
                fetch(next, j + 1);
                f32x4 s[RT][P];
                // Two pages' chains of products at a time, each of which would wait for itself.
#pragma unroll
                for (int i0 = 0; i0 < P; i0 += 2) {
#pragma unroll
                    for (int w = 0; w < 4; w++)
#pragma unroll
                        for (int i = i0; i < i0 + 2; i++) {
                            const f16x8 kf = as_f16x8(mx_decode8(at.kc[i][w], mx_scale(at.ks[i])));
#pragma unroll
                            for (int r = 0; r < RT; r++)
                                s[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, as_f16x8(qf[r][w]), w == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : s[r][i], 0, 0, 0);
                        }
                }
                const int key0 = (page_base + (wave + j * W) * P) * kPage;
                if (key0 + P * kPage - 1 > min_top) {  // some row does not see all of these keys
#pragma unroll
                    for (int i = 0; i < P; i++)
#pragma unroll
                        for (int v = 0; v < 4; v++) {
                            const int key = key0 + i * kPage + 4 * g + v;
#pragma unroll
                            for (int r = 0; r < RT; r++) s[r][i][v] = key <= my_top[r] ? s[r][i][v] : -INFINITY;
                            // Keys that no row sees may hold anything: their scales are taken as 2^-127, their values so as 0.
                            if (key > max_top) at.vs[i] &= ~(0xffu << (8 * v));
                        }
                }
                f16x8 wh[RT][P / 2];
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    float top = s[r][0][0];
#pragma unroll
                    for (int i = 0; i < P; i++)
#pragma unroll
                        for (int v = 0; v < 4; v++) top = fmaxf(top, s[r][i][v]);
                    top = top * p.scale_log2;
                    if (__builtin_amdgcn_ballot_w64(top - m[r] > kMostExponent)) {  // seldom: the reference moves
                        const float row_top = groups_max(top);
                        const bool grow = row_top - m[r] > kMostExponent;
                        const float reference = below(row_top, kMostExponent - kLazy);
                        const float corr = grow ? exp2_hw(m[r] - reference) : 1.0f;  // 0 from a row that had seen nothing
                        m[r] = grow ? reference : m[r];
                        l[r] = l[r] * corr;
#pragma unroll
                        for (int t = 0; t < 8; t++) o[r][t] = o[r][t] * corr;
                    }
                    float mul = p.scale_log2, add = -m[r];
                    if (const bool far = fabsf(add) >= kFar; __builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
                        for (int i = 0; i < P; i++)
#pragma unroll
                            for (int v = 0; v < 4; v++) s[r][i][v] = far ? s[r][i][v] * mul + add : __builtin_fmaf(s[r][i][v], mul, add);
                        mul = 1.0f, add = 0.0f;
                    }
                    const f16x2 ones = {static_cast<f16>(1.0f), static_cast<f16>(1.0f)};
#pragma unroll
                    for (int i = 0; i < P; i++) {
#pragma unroll
                        for (int v = 0; v < 4; v++) wh[r][i / 2][i % 2 * 4 + v] = static_cast<f16>(exp2_hw(__builtin_fmaf(s[r][i][v], mul, add)));
#pragma unroll
                        for (int v = 0; v < 4; v += 2)
                            l[r] = __builtin_amdgcn_fdot2(f16x2{wh[r][i / 2][i % 2 * 4 + v], wh[r][i / 2][i % 2 * 4 + v + 1]}, ones, l[r], false);
                    }
                }
#pragma unroll
                for (int i = 0; i < P; i += 2) {
                    // Dims 2 b and 2 b + 1 of the lane's eight are byte b of its keys' words.
                    auto pair = [&](auto byte) {
                        constexpr int b = decltype(byte)::value;
                        uint32_t x[2][4];  // [page][key % 4]
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int v = 0; v < 4; v++)
                                x[h][v] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(at.vc[i + h][v], mx_scale(at.vs[i + h], v), b));
#pragma unroll
                        for (int odd = 0; odd < 2; odd++) {
                            const uint32_t sel = odd ? 0x07060302u : 0x05040100u;  // high or low halves of two keys
                            const u32x4 vt = {__builtin_amdgcn_perm(x[0][1], x[0][0], sel), __builtin_amdgcn_perm(x[0][3], x[0][2], sel),
                                              __builtin_amdgcn_perm(x[1][1], x[1][0], sel), __builtin_amdgcn_perm(x[1][3], x[1][2], sel)};
#pragma unroll
                            for (int r = 0; r < RT; r++)
                                o[r][2 * b + odd] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(vt), wh[r][i / 2], o[r][2 * b + odd], 0, 0, 0);
                        }
                    };
                    pair(std::integral_constant<int, 0>{}), pair(std::integral_constant<int, 1>{});
                    pair(std::integral_constant<int, 2>{}), pair(std::integral_constant<int, 3>{});
                }
            };
            Step one, two;
            fetch(one, 0);
            __builtin_amdgcn_s_setprio(0);
            for (int j = 0; j < n; j += 2) {
                consume(one, two, j);
                if (j + 1 >= n) break;
                consume(two, one, j + 1);
            }
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int r = 0; r < RT; r++) l[r] = groups_sum(l[r]);

        // The row's place in out.
        auto at_of = [&](int row) {
            return static_cast<int64_t>(t0 + (row0 + row) / p.G) * p.n_heads + kvh * p.G + (row0 + row) % p.G;
        };
        float *const red_m = lds + W * kRows * kRowPitch, *const red_l = red_m + W * kRows;
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
        const bool whole = part.whole();
        const Partials<kRows> mine(p, parts.slot(kvh, worker, part.x == part.a));
        for (int i = tid; i < nrows * 16; i += kThreads) {
            const int row = i / 16, dim = i % 16 * 8;
            float M = kNoKeys, L = 0.0f, x[8] = {};
#pragma unroll
            for (int w = 0; w < W; w++) M = fmaxf(M, red_m[w * kRows + row]);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float part = red_l[w * kRows + row], f = filled(part) ? exp2_hw(red_m[w * kRows + row] - M) : 0.0f;
                L = L + part * f;
                const float *const src = lds + (w * kRows + row) * kRowPitch + dim;
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = x[e] + src[e] * f;
            }
            if (whole) store_piece(p.out + at_of(row) * D + dim, x, L);
            else {
                mine.put4(row, dim, f32x4{x[0], x[1], x[2], x[3]});
                mine.put4(row, dim + 4, f32x4{x[4], x[5], x[6], x[7]});
                if (dim == 0) mine.put_ml(row, M, L);
            }
        }
        if (!whole) {
            int from, to;
            parts.holders(part, from, to);
            if (last_of(p.counters + kvh * p.workers + from, to - from + 1, last))
                merge_partials<kRows, kThreads>(p, to - from + 1, nrows, lds, [&](int k) { return parts.slot(kvh, from + k, k == 0); }, at_of);
        }
    }
}

// ---- many rows: key blocks shared in LDS ----

// 128 rows a work-group; wave w owns rows 32 w .. + 31 of the tile, lane l = 32 h + c serves row c.
//
// Bound by the matrix unit (48% of the cycles), the VALU (softmax, conversion: 47%) and LDS (59%) in turns: each product
// reads a KiB of LDS, so four SIMDs at products take all of its 128 bytes a cycle, and the two waves of a SIMD mostly do
// the same. Tried against 233 us for 2000 tokens behind 12,000: group 1 half a step behind group 0, its softmax beside the
// other's products, 247; work-groups of one key group, two to a CU, 237; a wave's priority raised during its products 230
// (kept); keys staged 16 to a quarter wave, without bank conflicts, 229 (kept); group 0 always before group 1, by priority,
// 233 to 241; the two halves' chains of score products alternating 229.
// Measured, 16 heads on 8 kv heads: 2000 tokens behind 12,000 212 to 222 us by box (960 to 1,000 TFLOP/s), 4 of up to 512
// behind 900 to 3000 41 (490 TFLOP/s; of 256 to 512 50), 512 alone 16.
//
//   S^T = K Q^T   v_mfma_f32_32x32x16_f16: lane l ends with row c's scores of keys 8 (i / 4) + 4 h + i % 4 of each
//                 32-key half, so a row lives in two lanes.
//   O^T += V^T P^T  the lane's scores, as weights, are the B operand as they stand; the A operand, the same keys of dim
//                 c, comes from the transposing LDS read (lane r of 16 reads four dims of key r / 4).
// A block of 64 keys is converted once for all rows: a page a wave, on its way into LDS, a block ahead. KG groups of 4
// waves have the same rows and take the blocks in turn, each through buffers of its own; the others hand their
// partials to group 0.
constexpr int kTileRows = 128, kTileWaves = 4, kTileThreads = kTileWaves * kWave;
constexpr int kBlockPages = 4, kBlockKeys = kBlockPages * kPage;
static_assert(kBlockPages == kTileWaves);
// LDS rows, halves: keys on 68 dwords, values on 80, for reads without bank conflicts.
constexpr int kKeyRow = kHeadDim + 8, kValueRow = kHeadDim + 32;
constexpr int kKeyBuffer = kBlockKeys * kKeyRow, kValueBuffer = kBlockKeys * kValueRow;
typedef __fp16 tr16x4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __attribute__((address_space(3))) tr16x4 lds_tr16x4;
constexpr int kValuesAhead = 4;  // value operands in flight ahead of their products

// A row's half in a lane: element i is dims 8 i .. + 3 from dst on.
template <int N>
__device__ __forceinline__ void store_tile_row(f16 *dst, const f32x4 (&x)[N], float l) {
    const float inv = filled(l) ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        f16x4 y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = static_cast<f16>(x[i][e] * inv);
        *reinterpret_cast<f16x4 *>(dst + 8 * i) = y;
    }
}

// Joins n partials of a tile, slot_of(0) .. slot_of(n - 1) in that order, as the lanes that wrote them hold them; each
// group takes its part of the dims.
template <int KG, typename Slot>
__device__ __forceinline__ float merge_tiles(const Kv4Params &p, int n, int wave, int lane, int group, Slot slot_of, f32x4 (&x)[16 / KG]) {
    constexpr int N = 16 / KG;
    const int row = 32 * wave + lane % 32;
    float M = kNoKeys, L = 0.0f;
    for (int k = 0; k < n; k++) M = fmaxf(M, Partials<kTileRows>(p, slot_of(k)).get_ml(row).x);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
    for (int k = 0; k < n; k++) {
        const Partials<kTileRows> from(p, slot_of(k));
        const float2 ml = from.get_ml(row);
        u32x4 part[N];
#pragma unroll
        for (int i = 0; i < N; i++) part[i] = from.get_lane(wave, group * N + i, lane);
        const float w = filled(ml.y) ? exp2_hw(ml.x - M) : 0.0f;
        L = L + ml.y * w;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[i][e] = x[i][e] + __uint_as_float(part[i][e]) * w;
    }
    return L;
}

template <int KG>
__global__ void __launch_bounds__(KG *kTileThreads, 2) kv4_tile_kernel(Kv4Params p) {
    constexpr int D = kHeadDim;
    __shared__ __align__(16) f16 lds[KG * 2 * (kKeyBuffer + kValueBuffer)];
    __shared__ bool last;
    const int group = KG == 1 ? 0 : uniform(static_cast<int>(threadIdx.x) / kTileThreads);
    const int tid = static_cast<int>(threadIdx.x) % kTileThreads, lane = tid % kWave, wave = uniform(tid / kWave);
    f16 *const k_lds = lds + group * 2 * kKeyBuffer, *const v_lds = lds + KG * 2 * kKeyBuffer + group * 2 * kValueBuffer;
    const int h = lane >> 5, c = lane & 31;
    const int kvh = static_cast<int>(blockIdx.x) % p.n_kv;
    const int worker = static_cast<int>(blockIdx.x) / p.n_kv;
    const uint8_t *const pool = p.pool + kvh * kKv4Page;
    const uint32_t block_bytes = static_cast<uint32_t>(p.n_kv) * kKv4Page;
    const int table_top = p.max_blocks * kPage - 1;

    // A work-group an entry: the tiles with most keys first.
    Parts<kTileRows, kBlockKeys> parts(p, lane, p.workers > 0 ? worker : worker % p.S * p.tiles + p.tiles - 1 - worker / p.S);
    Part part;
    while (parts.next(part)) {
        const int t0 = part.t0, rows = part.rows, row0 = part.tile * kTileRows;
        const int32_t *const table = p.tables + static_cast<int64_t>(part.seq) * p.max_blocks;
        // Positions count up, so first and last rows bound them. Rows past the last repeat it.
        auto top_of = [&](int row) { return min(max(p.positions[t0 + min(row, rows - 1) / p.G], -1), table_top); };
        const int my_row = min(row0 + 32 * wave + c, rows - 1);
        const bool mine = row0 + 32 * wave + c < rows;
        const int my_tok = t0 + my_row / p.G, my_head = kvh * p.G + my_row % p.G;
        f16x8 qf[8];
        {
            const f16 *const qp = p.q + my_tok * p.q_stride + my_head * D;
#pragma unroll
            for (int i = 0; i < 8; i++) qf[i] = *reinterpret_cast<const f16x8 *>(qp + 16 * i + 8 * h);
        }
        int my_top = top_of(my_row), lo_top = uniform(top_of(row0 + 32 * wave));  // of the row, of the wave
        const int max_top = uniform(top_of(row0 + kTileRows - 1));                // of the tile
        const int all_pages = (max_top + kPage) / kPage, all_blocks = (all_pages + kBlockPages - 1) / kBlockPages;
        const int block0 = (part.x - part.a) << p.shift, block1 = part.stop == part.b ? all_blocks : min((part.stop - part.a) << p.shift, all_blocks);
        const int pages = min(all_pages, block1 * kBlockPages), blocks = max(block1 - block0, 0);
        my_top = min(my_top, block1 * kBlockKeys - 1), lo_top = min(lo_top, block1 * kBlockKeys - 1);  // a group may step past the part

        float m = -INFINITY, l = 0.0f;
        f32x16 o[4];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] = 0.0f;

        // Step b of this group is block block0 + b KG + group; its page of this wave. The ids of 64 steps' pages, one a lane.
        auto page_of = [&](int b) { return (block0 + b * KG + group) * kBlockPages + wave; };
        auto id_of = [&](int b) {
            const int page = page_of(b);
            return page < pages ? table[page] : -1;
        };
        int ids = -1, next_ids = id_of(lane);
        u32x4 kr, vr;
        uint32_t ks, vs;
        auto fetch = [&](int b) {
            if (b % kWave == 0) {
                ids = next_ids;
                next_ids = id_of(b + kWave + lane);
            }
            const uint32_t block = __builtin_amdgcn_readlane(ids, b % kWave);
            const bool ok = block < static_cast<uint32_t>(p.num_blocks);  // else no records: the loads give zeros
            const auto d = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(pool) + static_cast<uint64_t>(ok ? block : 0) * block_bytes, 0,
                                                             ok ? kKv4Page : 0, kDescWord3);
            kr = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(d, kHeadDim / 2 * (lane % 16) + 16 * (lane / 16), 0, 0));  // key l % 16, dims 32 (l / 16) ..
            ks = __builtin_amdgcn_raw_buffer_load_b8(d, kKv4KeyScales + 4 * (lane % 16) + lane / 16, 0, 0);
            vr = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(d, kKv4Values + 16 * lane, 0, 0));
            vs = __builtin_amdgcn_raw_buffer_load_b32(d, kKv4ValueScales + kPage * (lane % 16 / 4) + 4 * (lane / 16), 0, 0);
        };
        auto stage = [&](int b) {
            f16 *const kp = k_lds + (b & 1) * kKeyBuffer + (kPage * wave + lane % 16) * kKeyRow + 32 * (lane / 16);
            f16 *const vp = v_lds + (b & 1) * kValueBuffer + (kPage * wave + 4 * (lane / 16)) * kValueRow + 8 * (lane % 16);
            const int key0 = page_of(b) * kPage + 4 * (lane / 16);
            if (page_of(b) * kPage + kPage - 1 > max_top)
#pragma unroll
                for (int v = 0; v < 4; v++)  // keys that no row sees may hold anything: their values are read as 0
                    if (key0 + v > max_top) vs &= ~(0xffu << (8 * v));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                *reinterpret_cast<u32x4 *>(kp + 8 * i) = mx_decode8(kr[i], mx_scale(ks));
                *reinterpret_cast<u32x4 *>(vp + i * kValueRow) = mx_decode8(vr[i], mx_scale(vs, i));
            }
        };
        const int steps = (blocks + KG - 1) / KG;
        __syncthreads();  // the buffers' last readers, of the part before this
        if (steps > 0) {
            fetch(0);
            stage(0);
        }
        __syncthreads();
        for (int b = 0; b < steps; b++) {
            if (b + 1 < steps) fetch(b + 1);
            const f16 *const kl = k_lds + (b & 1) * kKeyBuffer + c * kKeyRow + 8 * h;
            const f16 *const vl = v_lds + (b & 1) * kValueBuffer + (4 * h + lane % 16 / 4) * kValueRow + 16 * (lane / 16 % 2) + 4 * (lane % 4);
            // Scores: the operands of a 32-key half are all requested before its first product, and each is
            // replaced by the other half's as soon as its product is issued.
            __builtin_amdgcn_s_setprio(1);
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
            f16x8 va[kValuesAhead];
#pragma unroll
            for (int n = 0; n < kValuesAhead; n++) va[n] = value(n);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            const int key0 = (block0 + b * KG + group) * kBlockKeys;
            if (key0 + kBlockKeys - 1 > lo_top) {  // some row of the wave does not see all of these keys
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[t][i] = key0 + 32 * t + 8 * (i / 4) + 4 * h + i % 4 <= my_top ? s[t][i] : -INFINITY;
            }
            float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
            for (int i = 1; i < 16; i++) top = fmaxf(fmaxf(top, s[0][i]), s[1][i]);
            top = top * p.scale_log2;
            if (__builtin_amdgcn_ballot_w64(top - m > kMostExponent)) {  // seldom: the reference moves
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
                for (int i = 0; i < 8; i++) w[j][i] = static_cast<f16>(exp2_hw(__builtin_fmaf(s[j / 2][8 * (j % 2) + i], mul, neg)));
#pragma unroll
                for (int i = 0; i < 4; i++) l = __builtin_amdgcn_fdot2(f16x2{w[j][2 * i], w[j][2 * i + 1]}, ones, l, false);
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int n = 0; n < 16; n++) {
                o[n % 4] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[n % kValuesAhead], w[n / 4], o[n % 4], 0, 0, 0);
                if (n + kValuesAhead < 16) va[n % kValuesAhead] = value(n + kValuesAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            if (b + 1 < steps) stage(b + 1);
            __syncthreads();
        }

        if constexpr (KG == 2) {  // group 1's partial, through the buffers (every wave is past its last block)
            f32x4 *const hand = reinterpret_cast<f32x4 *>(lds) + tid;
            static_assert(17 * kTileThreads * sizeof(f32x4) <= sizeof lds);
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
        }
        f16 *const dst = p.out + (static_cast<int64_t>(my_tok) * p.n_heads + my_head) * D + 4 * h;
        if (group == 0) {
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
            l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
            if (mine) {
                f32x4 x[16];
#pragma unroll
                for (int i = 0; i < 16; i++) x[i] = f32x4{o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1], o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]};
                if (part.whole()) {
                    store_tile_row(dst, x, l);
                } else {
                    const Partials<kTileRows> to(p, parts.slot(kvh, worker, part.x == part.a));
#pragma unroll
                    for (int i = 0; i < 16; i++) to.put_lane(wave, i, lane, x[i]);
                    if (h == 0) to.put_ml(32 * wave + c, filled(l) ? m : kNoKeys, l);
                }
            }
        }
        if (!part.whole()) {
            int from, to;
            parts.holders(part, from, to);
            if (last_of(p.counters + kvh * p.workers + from, to - from + 1, last) && mine) {
                constexpr int N = 16 / KG;
                f32x4 x[N];
                const float L = merge_tiles<KG>(p, to - from + 1, wave, lane, group, [&](int k) { return parts.slot(kvh, from + k, k == 0); }, x);
                store_tile_row(dst + 8 * N * group, x, L);
            }
        }
    }
}

// ---- host ----

constexpr int64_t kMostLaunch = UINT32_MAX / kThreads;  // HIP's bound on a launch's threads
constexpr int kMostSequences = 4096;                    // of a launch: a lane for each 64 of them
constexpr int kCus = 256;
constexpr int kWalkGroups = 2 * kCus;  // that share out a long context

// The workspace: the counters, at the same place whatever shape a call has, as they have to be 0 for the next one, which
// may be of another; then its partials.
constexpr int64_t kCounterBytes = kWalkGroups * static_cast<int64_t>(sizeof(uint32_t));

struct Plan {
    int rows;       // of a work-group: 16, 32 or 128
    int tiles;      // entries of a sequence
    int workers;    // work-groups of a kv head that share out its items; 0: one an entry
    int64_t bytes;  // of the workspace, with which items may be cut
    int64_t keys;   // of the longest context
};

int64_t bytes_of(const Plan &l, int n_kv) {
    return kCounterBytes + static_cast<int64_t>(l.workers) * n_kv * 2 * l.rows * (kHeadDim + 2) * static_cast<int64_t>(sizeof(float));
}

// Whether the work-groups share the items out evenly, or take one each. Sharing costs a scan of the lengths, partials
// and their merge; not sharing, the wait for the longest item.
//   Few rows: a work-group of its own takes 64 keys a wave in 0.95 us, all of them together 6.9 TB/s. Measured, us, one
//   each and shared: 1 sequence of 4000 keys 19.1, 10.7; of 131,000 477, 32; 4 of up to 3000 16.0, 13.5; 8 of 1000 9.2,
//   9.9; 32 of up to 4096 21.4, 24.4; 8 of up to 131,000 444, 124.
//   Tiles: a CU takes 64 keys of one in 0.85 us; shared, 6% more, and 15 us. Of several sequences only the longest context
//   is known: the others' are taken as half of it. Measured, us, one each and shared: 256 tokens behind 30,000 410, 76;
//   2 x 128 behind 4000 63.4, 33.8; 8 of up to 512 behind up to 8000 209, 117; 16 of up to 512 behind up to 9000 281, 190;
//   8 of up to 100 behind 500 to 3000 48.6, 44.5; 2 x 200 behind 1000 26.5, 27.9; 4 x 512 behind 900 to 3000 59.3, 61.6;
//   2000 behind 12,000 (an item a CU) 218, 226; 40 x 512 (8 items a CU) 342, 355.
bool share_out(bool tiled, bool alike, double items, int64_t keys) {
    const double steps = static_cast<double>((keys + 63) / 64);
    if (!tiled) return steps / kWaves * 0.95 > items * steps * 0.00126 + 7.0;
    const double load = items / kCus;
    const double one_each = alike ? std::max(1.0, std::ceil(load)) : std::max(1.0, 0.5 * load + 0.5);
    return steps * 0.85 * (one_each - 1.06 * (alike ? load : 0.5 * load)) > 15.0;
}

Plan plan(const EmberKv4AttnArgs &a, int64_t most, int sequences, int tokens) {
    const EmberRaggedBatch &b = a.batch;
    Plan l{};
    l.rows = most <= 16 ? 16 : most <= 32 ? 32 : kTileRows;
    l.tiles = static_cast<int>(std::clamp<int64_t>((most + l.rows - 1) / l.rows, 1, std::max(1, kMostSequences / sequences)));
    const int64_t keys = l.keys = std::min<int64_t>(a.max_context, static_cast<int64_t>(b.max_blocks) * kPage);
    const bool tiled = l.rows == kTileRows;
    // An item in more than 32 pieces is merged slower than it is read (131,000 keys in 64 pieces 36.6 us, in 32 32.4).
    const int most_workers = (tiled ? kCus : kWalkGroups) / b.n_kv;  // of kv heads that fill the chip by themselves, none
    double items = static_cast<double>(sequences) * l.tiles;
    if (tiled)  // of a tile a sequence, half is taken as empty; without tokens: the fewest items there may be
        items = tokens == 0 ? 0.0 : std::min(items, static_cast<double>(tokens) * (b.n_heads / b.n_kv) / l.rows + 0.5 * sequences);
    if (share_out(tiled, sequences == 1, b.n_kv * items, keys))
        l.workers = tiled ? most_workers : std::min(most_workers, 32 * sequences);
    if (l.workers > 0) l.bytes = bytes_of(l, b.n_kv);
    return l;
}

int64_t most_rows(const EmberRaggedBatch &b) { return static_cast<int64_t>(std::min(b.max_query, b.T)) * (b.n_heads / b.n_kv); }

// A step of prompt chunks and many more decodes is two launches, a form each: sequences of few rows are walked, the
// others' tiles shared out, an entry a sequence. It is told by the mean of the rows being less than a quarter of the most,
// and pays where the decodes as tiles, of half the longest context, would take the CUs 12.5 us. Measured, us, 8 kv heads,
// as tiles and as two launches: 960 decodes and 40 x 512 behind up to 1000 564, 346; 196 and 4 behind up to 4000 394, 210;
// 64 and 1 behind up to 3000 105, 66, 24 and 1 53.5, 49.0, 18 and 1 47.7, 48.5, 8 and 1 37, 43; 30 and 2 behind up to 2000
// 84, 58; 24 and 1 behind up to 600 26, 35.
// Few rows are 16, or 32 where one token has more than 16; none where a token has more than 32, whose decodes are tiles.
// Measured with 20 heads a kv head, all as tiles behind a first launch of no rows, and so: 200 decodes and 4 x 512 behind up
// to 4000 964, 845 (2 kv heads 272, 236), 64 and 1 behind up to 3000 226, 189, 30 and 2 behind up to 2000 188, 191.
int few_rows(int G) { return G <= 16 ? 16 : G <= 32 ? 32 : 0; }

bool mixed(const EmberKv4AttnArgs &a, int64_t most) {
    const EmberRaggedBatch &b = a.batch;
    if (most <= 32 || 4 * static_cast<int64_t>(b.T) * (b.n_heads / b.n_kv) >= b.S * most) return false;
    const double keys = static_cast<double>(std::min<int64_t>(a.max_context, static_cast<int64_t>(b.max_blocks) * kPage));
    return static_cast<double>(b.S) * b.n_kv * 0.5 * (keys / 64) * 0.85 / kCus > 12.5;
}

Plan shared_tiles(const EmberRaggedBatch &b) {
    Plan l{kTileRows, 1, kCus / b.n_kv, 0, 0};
    if (l.workers > 0) l.bytes = bytes_of(l, b.n_kv);
    return l;
}

// More items than CUs, each with a work-group, are dealt by length, which costs each of them a look at all lengths, 1 us
// for 64 sequences, 3 for 256: worth it where the longest are long. Measured, us, as they come and dealt: 48 sequences
// of 256 to 4095 keys 34.4, 28.0; 64 37.3, 31.4; 100 55.5, 47.0; 250 of 100 to 4000 101, 94; 64 of up to 4096 with up to
// 5 tokens 36.5, 33.6; 200 of up to 2000 45.2, 47.4; 64 of 2000 each 27.6, 28.5; 33 of up to 4095 23.5, 25.5.
bool dealt(const Plan &l, int n_kv, int sequences) {
    const int64_t items = static_cast<int64_t>(sequences) * l.tiles * n_kv, chunks = (sequences + kWave - 1) / kWave;
    return l.rows < kTileRows && l.workers == 0 && sequences <= kMostDealt && 4 * items > 5 * kCus && l.keys > 1536 + 512 * chunks;
}

// A launch: its form, without workers where the workspace does not let it share, and the rows that its sequences have.
struct Launch {
    Plan plan;
    int least, most;
};

// The launches of a call for `sequences` of its sequences.
int launches(const EmberKv4AttnArgs &a, int sequences, Launch (&out)[2]) {
    const EmberRaggedBatch &b = a.batch;
    const int64_t most = most_rows(b);
    auto can = [&](const Plan &l) { return l.workers > 0 && b.workspace && b.workspace_bytes >= l.bytes; };
    auto launch = [&](Plan l, int least, int rows) {
        if (!can(l)) l.workers = 0;  // uncut, an item each is as good
        return Launch{l, least, rows};
    };
    if (!mixed(a, most)) {
        out[0] = launch(plan(a, most, sequences, b.T), 1, INT_MAX);
        return 1;
    }
    const Plan shared = shared_tiles(b);
    const int few = few_rows(b.n_heads / b.n_kv);
    int n = 0;
    if (few > 0) out[n++] = launch(plan(a, few, sequences, b.T), 1, few);
    out[n++] = launch(can(shared) ? shared : plan(a, most, sequences, b.T), few + 1, INT_MAX);
    return n;
}

// One launch, for the sequences of p.
int run(const EmberRaggedBatch &b, Kv4Params p, const Launch &launch, hipStream_t stream) {
    const Plan &l = launch.plan;
    p.least = launch.least, p.most = launch.most;
    p.tiles = l.tiles;
    p.workers = l.workers;
    if (p.workers > 0) {
        const int64_t groups = static_cast<int64_t>(l.workers) * b.n_kv;
        p.counters = static_cast<uint32_t *>(b.workspace);
        p.part_acc = reinterpret_cast<float *>(static_cast<uint8_t *>(b.workspace) + kCounterBytes);
        p.part_ml = p.part_acc + 2 * groups * l.rows * kHeadDim;
    }
    const int64_t items = static_cast<int64_t>(p.S) * l.tiles * b.n_kv;
    const int64_t groups = p.workers > 0 ? static_cast<int64_t>(p.workers) * b.n_kv : items;
    if (groups > kMostLaunch)
        return set_error(EMBER_ERR_INVALID, "kv4_attn: too many work-groups for one launch (S %d x n_kv %d)", b.S, b.n_kv);
    if (l.rows == kTileRows) {
        // A work-group of two key groups fills a CU; with more items than CUs, one each, two to a CU.
        p.shift = 0;
        while ((static_cast<int64_t>(b.T) * p.G / kTileRows + items) * ((b.max_blocks / kBlockPages >> p.shift) + 2) > INT32_MAX) p.shift++;
        if (p.workers > 0 || items <= kCus)
            hipLaunchKernelGGL(kv4_tile_kernel<2>, dim3(static_cast<unsigned>(groups)), dim3(2 * kTileThreads), 0, stream, p);
        else
            hipLaunchKernelGGL(kv4_tile_kernel<1>, dim3(static_cast<unsigned>(groups)), dim3(kTileThreads), 0, stream, p);
        return EMBER_OK;
    }
    p.round = dealt(l, b.n_kv, p.S) ? std::max(1, kCus / b.n_kv) : 0;
    auto go = [&](auto kernel, int step_pages) {
        // The units of all items fit 31 bits.
        const int64_t most_items = static_cast<int64_t>(b.T) * p.G / l.rows + static_cast<int64_t>(p.S) * l.tiles;
        for (p.shift = 0; most_items * ((b.max_blocks / step_pages >> p.shift) + 2) > INT32_MAX; p.shift++) {}
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream, p);
    };
    // Steps of two pages leave room for a third work-group on a CU; where there is one at most, four pages are fewer
    // steps. Measured, us, two and four: 256 items of up to 4096 keys 23.2, 21.4; 512 35.7, 36.9; 2048 of up to 900
    // 32.4, 38.9.
    if (l.rows == 32) go(kv4_walk_kernel<2, kWaves, 2>, 2);
    else if (p.workers == 0 && items <= kCus) go(kv4_walk_kernel<1, kWaves, 4>, 4);
    else go(kv4_walk_kernel<1, kWaves, 2>, 2);
    return EMBER_OK;
}

}  // namespace

// Of these sizes and of smaller batches, which may be shared out where these are not, in any form of fewer rows, the more so
// the fewer their tokens. (From 16 sequences on a kv head has no more work-groups.)
int64_t kv4_workspace_bytes(const EmberKv4AttnArgs &a) {
    const int64_t most = most_rows(a.batch);
    int64_t bytes = a.batch.S > 1 && most > 32 ? shared_tiles(a.batch).bytes : 0;
    for (int64_t rows : {16, 32, 33})
        for (int sequences = 1; sequences <= std::min(a.batch.S, 16); sequences++)
            bytes = std::max(bytes, plan(a, std::min(most, rows), sequences, 0).bytes);
    return bytes;
}

int kv4_attn_plan(const EmberKv4AttnArgs &a, EmberKv4Launch *out) {
    Launch each[2];
    const int sequences = std::min(kMostSequences, a.batch.S), n = launches(a, sequences, each);
    for (int i = 0; i < n; i++) {
        const Plan &l = each[i].plan;
        out[i] = {l.bytes, l.rows, l.workers, dealt(l, a.batch.n_kv, sequences), each[i].least, each[i].most, 0};
    }
    return n;
}

int launch_kv4_attn(const EmberKv4AttnArgs &a, hipStream_t stream) {
    const EmberRaggedBatch &b = a.batch;
    Kv4Params p{};
    p.q = static_cast<const f16 *>(b.q), p.pool = static_cast<const uint8_t *>(b.k_cache), p.out = static_cast<f16 *>(b.out);
    p.positions = b.positions;
    p.q_stride = b.q_stride;
    p.T = b.T, p.max_blocks = b.max_blocks, p.n_heads = b.n_heads, p.n_kv = b.n_kv, p.G = b.n_heads / b.n_kv;
    p.num_blocks = b.num_blocks;
    p.scale_log2 = b.scale * kLog2e;
    for (int s0 = 0; s0 < b.S; s0 += kMostSequences) {
        p.S = std::min(kMostSequences, b.S - s0);
        p.query_start = b.query_start + s0, p.tables = b.block_tables + static_cast<int64_t>(s0) * b.max_blocks;
        Launch each[2];
        const int n = launches(a, p.S, each);
        for (int i = 0; i < n; i++)
            if (const int e = run(b, p, each[i], stream); e != EMBER_OK) return e;
    }
    return hip_status(hipGetLastError(), "kv4_attn");
}

}  // namespace ember::hip
