// A step's integers from its requests' lengths, on the device.
//
// With c_s tokens cached and n_s new, sequence s has h_s = ceil(c_s / 16)
// pages and needs d_s = ceil((c_s + n_s) / 16) - h_s more. Two running sums,
// of n (query_start, the tokens' rows) and of d (each sequence's run of the
// free list), give everything else entry by entry.
//
// One launch: every work-group takes the running sums of all S sequences
// (S <= 4096: loads that hit L2, one scan), then the work-groups share out the
// table entries and the tokens. Both sums stay below 2^31 (checked by the
// launcher), so one scan carries them as the halves of a 64-bit word. Only
// when the totals exceed the token rows or the free list does a second scan
// follow, of what the accepted sequences have.
//
// Bound by latency: 9 work-groups for 32 sequences take 6.2 us (lengths, scan,
// table entries wait for one another), 501 for 1000 sequences 9.9 us, of which
// the tables' 12.6 MB are 2 us. Tokens on work-groups of their own gained nothing.
//
// A request named twice would take two runs of pages for one row: a bitmap of
// the rows seen, and one of those seen again, find it, whatever order the
// atomics land in.
#include <algorithm>

#include "device.hpp"
#include "kernels.hpp"

namespace ember::hip {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kSegment = 1024;   // table entries of one row that a wave writes at a time
constexpr int kMaxGroups = 512;  // work-groups: two per CU

__device__ __forceinline__ uint64_t pack(int tokens, int pages) {
    return static_cast<uint64_t>(pages) << 32 | static_cast<uint32_t>(tokens);
}
__device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPage - 1) / kPage; }

// The sum of `own` over the threads before this one, and over the work-group.
__device__ __forceinline__ uint64_t scan_threads(uint64_t own, uint64_t *wave_sums, uint64_t &total) {
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    uint64_t x = own;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint64_t y = __shfl_up(x, o, kWave);
        x += lane >= o ? y : 0;
    }
    __syncthreads();  // an earlier scan's sums have been read
    if (lane == kWave - 1) wave_sums[wave] = x;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        before += w < wave ? wave_sums[w] : 0;
        total += wave_sums[w];
    }
    return before + x - own;
}

// VEC: table rows move 4 entries at a time (max_blocks a multiple of 4, both tables 16-byte aligned).
template <bool VEC>
__global__ void __launch_bounds__(kThreads) step_tables_kernel(EmberStepTablesArgs a) {
    // Per sequence: its request's row (-1: none), cached tokens, new tokens, first token row, first entry of the
    // free list. The last two are written after the bitmaps, which stand in their place, have been read.
    extern __shared__ int32_t lds[];
    __shared__ uint64_t wave_sums[kWaves];
    __shared__ int any_bits, longest;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    const int S = a.S, W = a.max_blocks;
    int32_t *const row_of = lds, *const cached = lds + S, *const fresh = lds + 2 * S;
    int32_t *const first_token = lds + 3 * S, *const first_free = lds + 4 * S;
    uint32_t *const seen = reinterpret_cast<uint32_t *>(lds + 3 * S);
    const int words = a.request ? (a.R + 31) / 32 : 0;
    uint32_t *const again = seen + words;
    const int cursor = a.free_cursor ? min(max(*a.free_cursor, 0), a.n_free) : 0;
    if (tid == 0) any_bits = longest = 0;
    for (int i = tid; i < 2 * words; i += kThreads) seen[i] = 0;
    __syncthreads();

    // Each sequence's request, lengths, and whether it can be in the step at all.
    // (four a thread at a time, so that their loads are out together)
    int bits = 0;
    for (int s0 = tid; s0 < S; s0 += 4 * kThreads) {
        int r[4], c[4], n[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int s = min(s0 + i * kThreads, S - 1);
            r[i] = a.request ? a.request[s] : s;
            n[i] = a.new_len[s];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = r[i] >= 0 && r[i] < a.R ? a.cached_len[r[i]] : -1;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int s = s0 + i * kThreads;
            if (s >= S) break;
            const bool ok = c[i] >= 0 && c[i] <= W * kPage && n[i] >= 0;
            const bool wide = ok && static_cast<int64_t>(c[i]) + n[i] > static_cast<int64_t>(W) * kPage;
            bits |= (ok ? 0 : EMBER_STEP_INVALID) | (wide ? EMBER_STEP_WIDE : 0);
            row_of[s] = ok ? r[i] : -1;
            cached[s] = ok ? c[i] : 0;
            fresh[s] = ok && !wide ? n[i] : 0;
            if (words && r[i] >= 0 && r[i] < a.R) {
                const uint32_t bit = 1u << (r[i] & 31);
                if (atomicOr(&seen[r[i] >> 5], bit) & bit) atomicOr(&again[r[i] >> 5], bit);
            }
        }
    }
    __syncthreads();
    if (words) {
        for (int s = tid; s < S; s += kThreads) {
            const int r = row_of[s];
            if (r < 0 || !(again[r >> 5] >> (r & 31) & 1)) continue;
            row_of[s] = -1;
            cached[s] = fresh[s] = 0;
            bits |= EMBER_STEP_INVALID;
        }
        __syncthreads();
    }

    // The running sums; a thread takes `per` sequences in a row.
    const int per = (S + kThreads - 1) / kThreads;
    const int s0 = min(tid * per, S), s1 = min(s0 + per, S);
    auto need_of = [&](int s) { return pages_of(cached[s] + fresh[s]) - pages_of(cached[s]); };
    uint64_t own = 0, total;
    for (int s = s0; s < s1; s++) own += pack(fresh[s], need_of(s));
    uint64_t at = scan_threads(own, wave_sums, total);
    const uint32_t rows = static_cast<uint32_t>(a.max_tokens), avail = static_cast<uint32_t>(a.n_free - cursor);
    if (static_cast<uint32_t>(total) > rows || static_cast<uint32_t>(total >> 32) > avail) {
        // The sums only grow: the sequences past the token rows are the last ones, and so are, of those that need
        // pages, the ones past the free list. Each is judged by the sums up to and with itself.
        own = 0;
        for (int s = s0; s < s1; s++) {
            const int need = need_of(s);
            at += pack(fresh[s], need);
            const bool late = static_cast<uint32_t>(at) > rows;
            const bool none = !late && need > 0 && static_cast<uint32_t>(at >> 32) > avail;
            bits |= (late ? EMBER_STEP_LATE : 0) | (none ? EMBER_STEP_SHORT : 0);
            if (late || none) fresh[s] = 0;
            else own += pack(fresh[s], need);
        }
        at = scan_threads(own, wave_sums, total);
    }
    int top = 0;
    for (int s = s0; s < s1; s++) {
        const int context = cached[s] + fresh[s];
        first_token[s] = static_cast<int32_t>(at);
        first_free[s] = cursor + static_cast<int32_t>(at >> 32);
        if (blockIdx.x == 0) {
            a.query_start[s] = static_cast<int32_t>(at);
            a.context_len[s] = context;
        }
        top = max(top, context);
        at += pack(fresh[s], need_of(s));
    }
    if (blockIdx.x == 0) {
        if (bits) atomicOr(&any_bits, bits);
        atomicMax(&longest, top);
    }
    __syncthreads();
    const int T = static_cast<int>(static_cast<uint32_t>(total));
    if (blockIdx.x == 0 && tid == 0) {
        a.query_start[S] = T;
        a.totals[0] = T;
        a.totals[1] = cursor + static_cast<int>(total >> 32);
        a.totals[2] = any_bits;
        a.totals[3] = longest;
    }

    // The table: a wave per row and segment of it. Pages taken by the step also go behind the request's own.
    const int segments = (W + kSegment - 1) / kSegment;
    for (int u = static_cast<int>(blockIdx.x) * kWaves + wave; u < (S + 1) * segments; u += static_cast<int>(gridDim.x) * kWaves) {
        const int s = u / segments, p0 = u % segments * kSegment, p1 = min(W, p0 + kSegment);
        int32_t *const dst = a.block_tables + static_cast<int64_t>(s) * W;
        const int row = s < S ? row_of[s] : -1;
        int32_t *const src = a.request_tables + static_cast<int64_t>(max(row, 0)) * W;
        const int have = row >= 0 ? pages_of(cached[s]) : 0, end = row >= 0 ? pages_of(cached[s] + fresh[s]) : 0;
        const int next = row >= 0 ? first_free[s] - have : 0;  // page p >= have is free_blocks[next + p]
        auto entry = [&](int p) {
            if (p < have) return src[p];
            if (p < end) return src[p] = a.free_blocks[next + p];
            return s == S && p == 0 ? a.pad_block : -1;
        };
        if constexpr (VEC) {
#pragma unroll 4
            for (int p = p0 + 4 * lane; p < p1; p += 4 * kWave) {
                int4 e;
                if (p + 4 <= have) e = *reinterpret_cast<const int4 *>(src + p);
                else if (p >= end && p > 0) e = make_int4(-1, -1, -1, -1);
                else e = make_int4(entry(p), entry(p + 1), entry(p + 2), entry(p + 3));
                *reinterpret_cast<int4 *>(dst + p) = e;
            }
        } else {
            for (int p = p0 + lane; p < p1; p += kWave) dst[p] = entry(p);
        }
    }

    // The tokens, one thread each: the last sequence that starts at or before the row (those without tokens start
    // where the next one does).
    for (int64_t t64 = static_cast<int64_t>(blockIdx.x) * kThreads + tid; t64 < a.max_tokens;
         t64 += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int t = static_cast<int>(t64);
        int s = S, pos = 0, block = a.pad_block;
        if (t < T) {
            int lo = 0, hi = S;  // first_token[lo] <= t; first_token[hi], were there one, is past t
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (first_token[mid] <= t) lo = mid;
                else hi = mid;
            }
            s = lo;
            pos = cached[s] + t - first_token[s];
            const int page = pos / kPage, have = pages_of(cached[s]);
            block = page < have ? a.request_tables[static_cast<int64_t>(row_of[s]) * W + page]
                                : a.free_blocks[first_free[s] + page - have];
        }
        a.positions[t] = pos;
        a.token_seq[t] = s;
        a.slots[t] = block >= 0 ? static_cast<int64_t>(block) * kPage + pos % kPage : -1;
    }
}

}  // namespace

hipError_t launch_step_tables(const EmberStepTablesArgs &a, hipStream_t stream) {
    const int words = a.request ? (a.R + 31) / 32 : 0;
    const size_t lds = sizeof(int32_t) * (3 * static_cast<size_t>(a.S) + 2 * static_cast<size_t>(std::max(a.S, words)));
    const int64_t units = static_cast<int64_t>(a.S + 1) * ((a.max_blocks + kSegment - 1) / kSegment);
    const int64_t groups = std::max((units + kWaves - 1) / kWaves, (static_cast<int64_t>(a.max_tokens) + kThreads - 1) / kThreads);
    const dim3 grid(static_cast<unsigned>(std::clamp<int64_t>(groups, 1, kMaxGroups)));
    const bool vec = a.max_blocks % 4 == 0 && (reinterpret_cast<uintptr_t>(a.request_tables) |
                                               reinterpret_cast<uintptr_t>(a.block_tables)) % 16 == 0;
    if (vec) hipLaunchKernelGGL(step_tables_kernel<true>, grid, dim3(kThreads), lds, stream, a);
    else hipLaunchKernelGGL(step_tables_kernel<false>, grid, dim3(kThreads), lds, stream, a);
    return hipGetLastError();
}

}  // namespace ember::hip
