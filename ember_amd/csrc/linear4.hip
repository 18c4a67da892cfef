// Linear layers with 4-bit weights, and the weights' preparation.
//
// C[M, N] = A[M, K] . W[N, K]^T on v_mfma_f32_16x16x32_f16: W is the A operand.
// A block of packed W is 16 features x 128 columns: lane 16 g + c holds, in 16
// bytes, feature c's columns 32 s + 8 g .. + 7 of its four steps s, a word each
// (four conversions); the feature's four scales are a word too. So W is read
// in whole KiB by the lanes that convert it and never shuffled, and the
// activations' lane reads its row's same columns, four lanes 64 bytes in one
// piece. (With a lane's 32 columns adjacent, one scale a lane, each load of
// activations touched 64 lines and not 16: 32 rows of 12288 x 2048 16.6 us.)
//
// A row's sum: wave w of 8 chains the blocks w, w + 8, ... in order, and the
// waves' sums are added in order, whatever M is and however many features a
// work-group takes. Hence the same bits for a row in any batch.
#include <algorithm>
#include <cfloat>

#include "four_bit.hpp"
#include "kernels.hpp"
#include "linear.hpp"

namespace ember::hip {
namespace {

constexpr int kBlockCols = 128;
constexpr int kBlockCodes = 16 * kBlockCols / 2;             // bytes
constexpr int kBlockBytes = kBlockCodes + 16 * kBlockCols / kMxGroup;
constexpr int kWaves4 = kLinearRuns;
constexpr int kThreads4 = kWaves4 * kWave;

__host__ __device__ constexpr int blocks_of(int K) { return (K + kBlockCols - 1) / kBlockCols; }

struct Gemv4Params {
    const f16 *A;
    const uint8_t *W;
    void *C;
    int64_t lda, ldc;
    int M, N, K;
    bool vec;  // C's rows take a lane's four features in one store
};

// A block of activations in LDS: [row][16 pieces of 16 bytes], piece p of row r
// at place p ^ (r % 16). Staged by lanes that read 256 bytes of a row side by
// side; read as the products' operand by 16 rows at a time, on all banks. Read
// straight from memory in the operand's order, every lane of a quad of lanes
// is on a line of its own, which costs four times the cycles of the lines.
constexpr int kStageTile = 16 * kBlockCols;  // halves of 16 rows

// Holds the compiler to the order of a stage's stores and of the reads by the wave's other lanes; no instruction.
__device__ __forceinline__ void own_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
}

// The four features n0 .. of a row, and what ADD_F32 adds them to.
template <int EP>
__device__ __forceinline__ f32x4 previous(const Gemv4Params &p, int row, int n0) {
    f32x4 old = {0.0f, 0.0f, 0.0f, 0.0f};
    if (EP != EMBER_EPILOGUE_ADD_F32 || row >= p.M) return old;
    const float *const at = static_cast<const float *>(p.C) + row * p.ldc + n0;
    if (p.vec && n0 + 3 < p.N) return *reinterpret_cast<const f32x4 *>(at);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n0 + i < p.N) old[i] = at[i];
    return old;
}

template <int EP>
__device__ __forceinline__ void finish(const Gemv4Params &p, int row, int n0, f32x4 sum, const f32x4 &old) {
    if (row >= p.M) return;
    const bool whole = p.vec && n0 + 3 < p.N;
    if constexpr (EP == EMBER_EPILOGUE_SILU_MUL) {  // gate rows even, up rows odd
        f16 *const at = static_cast<f16 *>(p.C) + row * p.ldc + n0 / 2;
        const f16x2 h = {static_cast<f16>(clamp_half(silu(sum[0]) * sum[1])), static_cast<f16>(clamp_half(silu(sum[2]) * sum[3]))};
        if (whole) {
            *reinterpret_cast<f16x2 *>(at) = h;
        } else {
            if (n0 < p.N) at[0] = h[0];
            if (n0 + 2 < p.N) at[1] = h[1];
        }
    } else if constexpr (EP == EMBER_EPILOGUE_STORE_F16) {
        f16 *const at = static_cast<f16 *>(p.C) + row * p.ldc + n0;
        f16x4 h;
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = static_cast<f16>(clamp_half(sum[i]));
        if (whole) {
            *reinterpret_cast<f16x4 *>(at) = h;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (n0 + i < p.N) at[i] = h[i];
        }
    } else {
        float *const at = static_cast<float *>(p.C) + row * p.ldc + n0;
        if constexpr (EP == EMBER_EPILOGUE_ADD_F32) sum = old + sum;
        if (whole) {
            *reinterpret_cast<f32x4 *>(at) = sum;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (n0 + i < p.N) at[i] = sum[i];
        }
    }
}

// Blocks wave + 8 u of K from `block0` on, of MT tiles of rows, as the products' operands in registers: x[u][m][s].
template <int MT, int BPW>
__device__ __forceinline__ void load_rows(const Gemv4Params &p, f16 *stage, int m0, int rows, int block0, int lane, f16x8 (&x)[BPW][MT][4]) {
    const int c = lane % 16, g = lane / 16;
    const f16 *const src = p.A + m0 * p.lda + 8 * c;
    f16x8 raw[BPW][4 * MT];
#pragma unroll
    for (int u = 0; u < BPW; u++) {
        const int col = (block0 + u * kWaves4) * kBlockCols;
#pragma unroll
        for (int i = 0; i < 4 * MT; i++)
            if (4 * i < rows) raw[u][i] = col + 8 * c < p.K ? *reinterpret_cast<const f16x8 *>(src + min(4 * i + g, rows - 1) * p.lda + col) : f16x8{};
    }
#pragma unroll
    for (int u = 0; u < BPW; u++) {
#pragma unroll
        for (int i = 0; i < 4 * MT; i++)
            if (4 * i < rows) *reinterpret_cast<f16x8 *>(stage + (4 * i + g) * kBlockCols + 8 * (c ^ (4 * i + g) % 16)) = raw[u][i];
        own_fence();
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const int row = min(16 * m + c, rows - 1);  // rows past the last repeat it
                x[u][m][s] = *reinterpret_cast<const f16x8 *>(stage + row * kBlockCols + 8 * ((4 * s + g) ^ row % 16));
            }
        own_fence();
    }
}

// MT tiles of 16 rows, BPW blocks of K a wave. The work-group loads its rows
// once, each wave its own columns as operands in registers, and walks over
// tiles of 16 features, the W of the next kDepth in flight. LONG: more of K than
// that; each tile goes over it in rounds, rows and all.
//
// Bound by a launch's three trips to memory where W is small (1 row of 4096 x
// 1024 3.0 us), by reading W where it is large (8 rows of 151936 x 1024 15.9 us,
// 5.5 TB/s, 19 where no cache holds any of W; 1 of 24576 x 4096 12.2, 4.4 TB/s),
// and between them by what a CU takes in, A and W (32 rows of 12288 x 2048 7.8
// us, 64 9.6; added into f32, 32 of 2048 x 2048 4.3, of 2048 x 6144 8.0). Many
// rows convert W once for 32 or 64 of them: 512 of 4096 x 4096 24.6 us (700
// TFLOP/s), 2048 of 12288 x 2048 110 (940).
template <int EP, int MT, int BPW, bool LONG>
__global__ void __launch_bounds__(kThreads4, MT * BPW <= 2 ? 4 : 2) gemv4_kernel(Gemv4Params p) {
    constexpr int kDepth = LONG || BPW >= 4 ? 1 : 4 / BPW;
    constexpr int kStageBytes = kWaves4 * MT * kStageTile * static_cast<int>(sizeof(f16));
    static_assert(2 * kWaves4 * MT * kWave * sizeof(f32x4) <= kStageBytes);  // two buffers of sums
    __shared__ __align__(16) unsigned char lds[kStageBytes];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int c = lane % 16, g = lane / 16;
    const int tiles = (p.N + 15) / 16, stride = static_cast<int>(gridDim.x);
    const int m0 = static_cast<int>(blockIdx.y) * (16 * MT), rows = min(p.M - m0, 16 * MT);
    const int blocks = blocks_of(p.K);
    f16 *const stage = reinterpret_cast<f16 *>(lds) + wave * MT * kStageTile;
    f32x4 *const red = reinterpret_cast<f32x4 *>(lds);

    u32x4 codes[kDepth][BPW];
    uint32_t scale[kDepth][BPW];
    auto fetch = [&](int slot, int tile, int block0) {
#pragma unroll
        for (int u = 0; u < BPW; u++) {
            const uint8_t *const at = p.W + (static_cast<int64_t>(min(tile, tiles - 1)) * blocks + min(block0 + u * kWaves4, blocks - 1)) * kBlockBytes;
            codes[slot][u] = *reinterpret_cast<const u32x4 *>(at + 16 * lane);
            scale[slot][u] = *reinterpret_cast<const uint32_t *>(at + kBlockCodes + 4 * c);
        }
    };
    const int first = static_cast<int>(blockIdx.x);
    f16x8 x[BPW][MT][4];
    if constexpr (!LONG) {
#pragma unroll
        for (int d = 0; d < kDepth; d++) {
            fetch(d, first + d * stride, wave);
            __builtin_amdgcn_sched_barrier(0);  // in the order that the products wait for them
        }
        load_rows<MT, BPW>(p, stage, m0, rows, wave, lane, x);
        __syncthreads();  // the stages are the sums' buffers
    }

    int turn = 0;
    auto product = [&](int d, int tile, bool more) {
        f32x4 acc[MT];
#pragma unroll
        for (int m = 0; m < MT; m++) acc[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int block0 = wave; block0 < blocks; block0 += BPW * kWaves4) {
            if constexpr (LONG) {
                fetch(d, tile, block0);
                load_rows<MT, BPW>(p, stage, m0, rows, block0, lane, x);
            }
#pragma unroll
            for (int u = 0; u < BPW; u++) {
                if (block0 + u * kWaves4 >= blocks) break;
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const f16x8 w = as_f16x8(mx_decode8(codes[d][u][s], mx_scale(scale[d][u], s)));
#pragma unroll
                    for (int m = 0; m < MT; m++) acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, x[u][m][s], acc[m], 0, 0, 0);
                }
            }
            if constexpr (!LONG) break;
        }
        if constexpr (LONG) __syncthreads();
        else if (more) fetch(d, tile + kDepth * stride, wave);
        f32x4 *const sums = red + (turn & 1) * kWaves4 * MT * kWave + lane;
#pragma unroll
        for (int m = 0; m < MT; m++) sums[(wave * MT + m) * kWave] = acc[m];
        // The waves take turns at the sums' rows.
        const int mine = (wave - turn) & (kWaves4 - 1);
        const int row = m0 + 16 * mine + c, n0 = 16 * tile + 4 * g;
        const f32x4 old = mine < MT ? previous<EP>(p, row, n0) : f32x4{};
        __syncthreads();
        if (mine < MT) {
            f32x4 sum = sums[mine * kWave];
#pragma unroll
            for (int v = 1; v < kWaves4; v++) sum = sum + sums[(v * MT + mine) * kWave];
            finish<EP>(p, row, n0, sum, old);
        }
        if constexpr (LONG) __syncthreads();
        turn++;
    };
    // Whole rounds have no way out between their tiles, so that the waits for W count the loads behind it.
    int tile0 = first;
    for (; tile0 + (kDepth - 1) * stride < tiles; tile0 += kDepth * stride)
#pragma unroll
        for (int d = 0; d < kDepth; d++) product(d, tile0 + d * stride, true);
#pragma unroll
    for (int d = 0; d < kDepth - 1; d++)
        if (tile0 + d * stride < tiles) product(d, tile0 + d * stride, false);
}

// Prompts: 16 MT rows x 16 FT features a work-group. Each wave takes its own
// blocks of K for all of them, so the waves stay apart up to the sums, with the
// next block's loads out during a block's products.
//
// Bound by what a CU takes in of A and W through L2, 43 GB/s: 512 rows of 2048
// x 6144 18.9 to 20.1 us (640 to 680 TFLOP/s; added into f32 the same), 2048
// 78.5 (660), 300 of 4096 x 12288 60.7 (500).
template <int EP, int MT, int FT>
__global__ void __launch_bounds__(kThreads4, 2) gemm4_kernel(Gemv4Params p) {
    constexpr int kStageBytes = kWaves4 * MT * kStageTile * static_cast<int>(sizeof(f16));
    constexpr int kSumBytes = kWaves4 * MT * 4 * kWave * static_cast<int>(sizeof(f32x4));  // of 4 tiles of features at a time
    static_assert(kSumBytes <= kStageBytes && FT % 4 == 0);
    __shared__ __align__(16) unsigned char lds[kStageBytes];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int c = lane % 16, g = lane / 16;
    const int tiles = (p.N + 15) / 16, tile0 = static_cast<int>(blockIdx.x) * FT;
    const int m0 = static_cast<int>(blockIdx.y) * (16 * MT), rows = min(p.M - m0, 16 * MT);
    const int blocks = blocks_of(p.K);
    f16 *const stage = reinterpret_cast<f16 *>(lds) + wave * MT * kStageTile;
    const f16 *const src = p.A + m0 * p.lda + 8 * c;

    u32x4 codes[FT];
    uint32_t scale[FT];
    f16x8 raw[4 * MT];
    auto fetch = [&](int b) {
        const int col = b * kBlockCols;
#pragma unroll
        for (int i = 0; i < 4 * MT; i++)
            if (4 * i < rows) raw[i] = col + 8 * c < p.K ? *reinterpret_cast<const f16x8 *>(src + min(4 * i + g, rows - 1) * p.lda + col) : f16x8{};
#pragma unroll
        for (int f = 0; f < FT; f++) {
            const uint8_t *const at = p.W + (static_cast<int64_t>(min(tile0 + f, tiles - 1)) * blocks + b) * kBlockBytes;
            codes[f] = *reinterpret_cast<const u32x4 *>(at + 16 * lane);
            scale[f] = *reinterpret_cast<const uint32_t *>(at + kBlockCodes + 4 * c);
        }
    };
    f32x4 acc[FT][MT];
#pragma unroll
    for (int f = 0; f < FT; f++)
#pragma unroll
        for (int m = 0; m < MT; m++) acc[f][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (wave < blocks) fetch(wave);
    for (int b = wave; b < blocks; b += kWaves4) {
#pragma unroll
        for (int i = 0; i < 4 * MT; i++)
            if (4 * i < rows) *reinterpret_cast<f16x8 *>(stage + (4 * i + g) * kBlockCols + 8 * (c ^ (4 * i + g) % 16)) = raw[i];
        own_fence();
        u32x4 now[FT];
        uint32_t now_scale[FT];
#pragma unroll
        for (int f = 0; f < FT; f++) now[f] = codes[f], now_scale[f] = scale[f];
        fetch(min(b + kWaves4, blocks - 1));
#pragma unroll
        for (int s = 0; s < 4; s++) {
            f16x8 x[MT];
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const int row = min(16 * m + c, rows - 1);
                x[m] = *reinterpret_cast<const f16x8 *>(stage + row * kBlockCols + 8 * ((4 * s + g) ^ row % 16));
            }
#pragma unroll
            for (int f = 0; f < FT; f++) {
                const f16x8 w = as_f16x8(mx_decode8(now[f][s], mx_scale(now_scale[f], s)));
#pragma unroll
                for (int m = 0; m < MT; m++) acc[f][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, x[m], acc[f][m], 0, 0, 0);
            }
        }
        own_fence();
    }
    f32x4 *const red = reinterpret_cast<f32x4 *>(lds) + lane;
#pragma unroll
    for (int f0 = 0; f0 < FT; f0 += 4) {
        __syncthreads();
#pragma unroll
        for (int f = 0; f < 4; f++)
#pragma unroll
            for (int m = 0; m < MT; m++) red[((wave * 4 + f) * MT + m) * kWave] = acc[f0 + f][m];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MT * 4 / kWaves4; i++) {
            const int at = wave + i * kWaves4, row = m0 + 16 * (at % MT) + c, n0 = 16 * (tile0 + f0 + at / MT) + 4 * g;
            const f32x4 old = previous<EP>(p, row, n0);
            f32x4 sum = red[at * kWave];
#pragma unroll
            for (int v = 1; v < kWaves4; v++) sum = sum + red[(v * 4 * MT + at) * kWave];
            finish<EP>(p, row, n0, sum, old);
        }
    }
}

// Which rows a work-group takes together: more of them read W less often, fewer of them read less of A into each CU. A
// launch is bound by what a CU takes in (A's rows through L2 at a rate below W's), so the one with the fewest bytes of
// both for the CU that has most. Measured, us, 16, 32 and 64 rows together: 64 rows of 4096 x 2048 6.04, 5.93, 8.02; of
// 12288 x 2048 9.70, 9.37, 10.80; of 151936 x 1024 57.6, 35.3, 31.4; of 24576 x 4096 31.0, 21.0 (64: too many registers).
constexpr int kCus = 256;

int row_tiles(int M, int tiles, int blocks, int most) {
    int best = 1;
    int64_t least = INT64_MAX;
    for (int mt = 1; mt <= most; mt *= 2) {
        const int64_t y = (M + 16 * mt - 1) / (16 * mt);
        const int64_t bytes = blocks * (static_cast<int64_t>(16 * mt) * kBlockCols * 2 + (tiles * y + kCus - 1) / kCus * kBlockBytes);
        if (bytes < least) least = bytes, best = mt;
    }
    return best;
}

template <int EP>
hipError_t run_gemv4(const EmberGemv4Args &a, hipStream_t stream) {
    constexpr bool f16_out = EP == EMBER_EPILOGUE_STORE_F16 || EP == EMBER_EPILOGUE_SILU_MUL;
    constexpr int lane_out = EP == EMBER_EPILOGUE_SILU_MUL ? 2 : 4;  // of a lane's features
    Gemv4Params p{static_cast<const f16 *>(a.A), static_cast<const uint8_t *>(a.W), a.C, a.lda, a.ldc, a.M, a.N, a.K, false};
    p.vec = a.ldc % lane_out == 0 && reinterpret_cast<uintptr_t>(a.C) % (lane_out * (f16_out ? 2 : 4)) == 0;
    const int tiles = (a.N + 15) / 16, blocks = blocks_of(a.K);
    auto go = [&](auto kernel, int mt, int wgs) {  // wgs: work-groups that a CU holds
        const int y = (a.M + 16 * mt - 1) / (16 * mt);
        const int most = std::max(1, kCus * wgs / y), each = (tiles + most - 1) / most;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((tiles + each - 1) / each), static_cast<unsigned>(y)), dim3(kThreads4), 0, stream, p);
    };
    const int bpw = (blocks + kWaves4 - 1) / kWaves4;
    // Prompts whose K leaves the rows of one tile in registers only, where W's conversion bounds the launch. Measured, us,
    // in registers against 32 rows x 64 or 128 features: 2048 x 6144, 128 rows 11.4, 12.5; 192 rows 16.5, 12.6; 512 rows
    // 30.1, 18.7. 4096 x 12288, 32 rows 18.0, 27.2; 64 rows 28.1, 26.1; 512 rows over 200, 60. Of 24576 x 4096, 384 rows
    // 92, 119: up to 4096 columns registers win with any number of rows.
    if ((bpw > 4 && a.M > 128) || (bpw > 8 && a.M > 48)) {
        const int y = (a.M + 31) / 32;
        auto go = [&](auto kernel, int ft) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((tiles + ft - 1) / ft), static_cast<unsigned>(y)), dim3(kThreads4), 0, stream, p);
        };
        // 64 features where that is one work-group a CU at most: 256 rows of 2048 x 6144 13.0 against 16.9 us, 384 rows 24.1, 17.8.
        if (static_cast<int64_t>(y) * ((tiles + 3) / 4) <= kCus) go(gemm4_kernel<EP, 2, 4>, 4);
        else go(gemm4_kernel<EP, 2, 8>, 8);
        return hipGetLastError();
    }
    // Rows in registers: at most 128 of them.
    const int mt = row_tiles(a.M, tiles, blocks, bpw <= 2 ? 4 : bpw <= 4 ? 2 : 1);
    if (bpw <= 1) {
        if (mt == 1) go(gemv4_kernel<EP, 1, 1, false>, 1, 2);
        else if (mt == 2) go(gemv4_kernel<EP, 2, 1, false>, 2, 2);
        else go(gemv4_kernel<EP, 4, 1, false>, 4, 1);
    } else if (bpw <= 2) {
        if (mt == 1) go(gemv4_kernel<EP, 1, 2, false>, 1, 2);
        else if (mt == 2) go(gemv4_kernel<EP, 2, 2, false>, 2, 1);
        else go(gemv4_kernel<EP, 4, 2, false>, 4, 1);
    } else if (bpw <= 4) {
        if (mt == 1) go(gemv4_kernel<EP, 1, 4, false>, 1, 1);
        else go(gemv4_kernel<EP, 2, 4, false>, 2, 1);
    } else if (bpw <= 8) {
        go(gemv4_kernel<EP, 1, 8, false>, 1, 1);
    } else {
        go(gemv4_kernel<EP, 1, 4, true>, 1, 2);
    }
    return hipGetLastError();
}

// A thread per 8 columns (one word of codes), in the order of the output. Once per weight: 151936 x 1024 72 us, 24576 x
// 4096 46 (2.3 TB/s read and written, half of a copy's rate: codes are read in
// pieces of 4 bytes and scales one by one, which is not worth more for a layout
// that a program does once).
__global__ void __launch_bounds__(256) gemv4_pack_kernel(const uint8_t *codes, const uint8_t *scales, int N, int K, uint8_t *out) {
    const int blocks = blocks_of(K);
    const int64_t words = static_cast<int64_t>((N + 15) / 16) * blocks * (kBlockCodes / 4);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < words; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int word = static_cast<int>(i % (kBlockCodes / 4)), lane = word / 4, s = word % 4;
        const int64_t block = i / (kBlockCodes / 4);
        const int64_t row = block / blocks * 16 + lane % 16, group = block % blocks * (kBlockCols / kMxGroup) + s;
        const bool real = row < N && group < K / kMxGroup;
        uint8_t *const dst = out + block * kBlockBytes;
        reinterpret_cast<uint32_t *>(dst)[word] = real ? reinterpret_cast<const uint32_t *>(codes + row * (K / 2) + group * (kMxGroup / 2))[lane / 16] : 0u;
        if (lane < 16) dst[kBlockCodes + 4 * lane + s] = real ? scales[row * (K / kMxGroup) + group] : 0;
    }
}

// A thread per 8 columns, four lanes a group. Bound by memory: 24576 x 4096 f16 49 us (5.2 TB/s), f32 80. Rows need no
// alignment, so elements are read one by one.
template <typename T>
__global__ void __launch_bounds__(256) mx_quantize_kernel(EmberMxQuantizeArgs a) {
    const int pieces = a.cols / 8;
    const int64_t all = static_cast<int64_t>(a.rows) * pieces;  // a multiple of 4: a quad has all of its lanes or none
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / pieces;
        const int col = static_cast<int>(i % pieces) * 8;
        const T *const src = static_cast<const T *>(a.x) + row * a.ld + col;
        float x[8], m = 0.0f, bad = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = to_f32(src[e]);
            bad = v != v ? 1.0f : bad;
            x[e] = fminf(fmaxf(v, -FLT_MAX), FLT_MAX);
            m = fmaxf(m, fabsf(x[e]));
        }
        m = fmaxf(m, dpp_mov<kDppQuadXor1>(m)), m = fmaxf(m, dpp_mov<kDppQuadXor2>(m));
        bad = fmaxf(bad, dpp_mov<kDppQuadXor1>(bad)), bad = fmaxf(bad, dpp_mov<kDppQuadXor2>(bad));
        const int byte = mx_scale_byte(m);
        *reinterpret_cast<uint32_t *>(a.codes + row * (a.cols / 2) + col / 2) = bad != 0.0f ? 0u : mx_encode8(x, mx_scale(byte));
        if (col % kMxGroup == 0) a.scales[row * (a.cols / kMxGroup) + col / kMxGroup] = bad != 0.0f ? 255 : static_cast<uint8_t>(byte);
    }
}

unsigned grid_for(int64_t threads) { return static_cast<unsigned>(std::min<int64_t>((threads + 255) / 256, 1 << 16)); }

}  // namespace

int64_t gemv4_packed_bytes(int N, int K) { return static_cast<int64_t>((N + 15) / 16) * blocks_of(K) * kBlockBytes; }

hipError_t launch_gemv4_pack(const uint8_t *codes, const uint8_t *scales, int N, int K, void *out, hipStream_t stream) {
    hipLaunchKernelGGL(gemv4_pack_kernel, dim3(grid_for(gemv4_packed_bytes(N, K) / 4)), dim3(256), 0, stream, codes, scales, N, K,
                       static_cast<uint8_t *>(out));
    return hipGetLastError();
}

hipError_t launch_mx_quantize(const EmberMxQuantizeArgs &a, hipStream_t stream) {
    const dim3 grid(grid_for(static_cast<int64_t>(a.rows) * (a.cols / 8)));
    if (a.dtype == EMBER_DTYPE_F16) hipLaunchKernelGGL(mx_quantize_kernel<f16>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(mx_quantize_kernel<float>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_gemv4(const EmberGemv4Args &all, hipStream_t stream) {
    constexpr int kMostRows = 1 << 20;  // of a launch, whose y counts at most 65535 tiles, of 32 rows where they are many
    const int64_t element = all.epilogue == EMBER_EPILOGUE_STORE_F16 || all.epilogue == EMBER_EPILOGUE_SILU_MUL ? sizeof(f16) : sizeof(float);
    for (int m0 = 0; m0 < all.M; m0 += kMostRows) {
        EmberGemv4Args a = all;
        a.M = std::min(all.M - m0, kMostRows);
        a.A = static_cast<const f16 *>(all.A) + m0 * all.lda;
        a.C = static_cast<uint8_t *>(all.C) + m0 * all.ldc * element;
        hipError_t e;
        switch (a.epilogue) {
            case EMBER_EPILOGUE_STORE_F16: e = run_gemv4<EMBER_EPILOGUE_STORE_F16>(a, stream); break;
            case EMBER_EPILOGUE_STORE_F32: e = run_gemv4<EMBER_EPILOGUE_STORE_F32>(a, stream); break;
            case EMBER_EPILOGUE_ADD_F32: e = run_gemv4<EMBER_EPILOGUE_ADD_F32>(a, stream); break;
            default: e = run_gemv4<EMBER_EPILOGUE_SILU_MUL>(a, stream); break;
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ember::hip
