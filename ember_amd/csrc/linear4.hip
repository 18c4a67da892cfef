// Linear layers with 4-bit weights, and the weights' preparation.
//
// C[M, N] = A[M, K] . W[N, K]^T on v_mfma_f32_16x16x32_f16: W is the A operand.
// A block of packed W is 16 features x 128 columns: lane 16 g + c holds
// feature c's columns 32 g .. + 31, one group with one scale, as 16 bytes.
// Step s of the block's four takes the lane's columns 8 s .. + 7 (one word,
// four conversions), and the activations' lane the same columns of its row:
// the order in which a product's columns are summed is free. So W is read in
// whole KiB by the lanes that convert it, once, and is never shuffled.
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

// MT tiles of 16 rows, FT tiles of 16 features.
template <int MT, int FT, int EP>
__global__ void __launch_bounds__(kThreads4)
    gemv4_kernel(const f16 *__restrict__ A, int64_t lda, const uint8_t *__restrict__ W, int M, int N, int K, void *__restrict__ C,
                 int64_t ldc) {
    __shared__ f32x4 red[kWaves4 * MT * FT * kWave];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % kWave, wave = uniform(tid / kWave);
    const int c = lane % 16, g = lane / 16;
    const int tile0 = static_cast<int>(blockIdx.x) * FT, tiles = (N + 15) / 16;
    const int m0 = static_cast<int>(blockIdx.y) * (16 * MT);
    const int blocks = blocks_of(K);
    const uint8_t *w[FT];
#pragma unroll
    for (int f = 0; f < FT; f++) w[f] = W + static_cast<int64_t>(min(tile0 + f, tiles - 1)) * blocks * kBlockBytes;
    const f16 *x[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) x[m] = A + static_cast<int64_t>(min(m0 + 16 * m + c, M - 1)) * lda + 32 * g;
    f32x4 acc[FT][MT];
#pragma unroll
    for (int f = 0; f < FT; f++)
#pragma unroll
        for (int m = 0; m < MT; m++) acc[f][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int b = wave; b < blocks; b += kWaves4) {
        u32x4 codes[FT];
        float scale[FT];
#pragma unroll
        for (int f = 0; f < FT; f++) {
            codes[f] = *reinterpret_cast<const u32x4 *>(w[f] + b * kBlockBytes + 16 * lane);
            scale[f] = mx_scale(w[f][b * kBlockBytes + kBlockCodes + lane]);
        }
        const bool inside = b * kBlockCols + 32 * g < K;
        f16x8 xv[MT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int s = 0; s < 4; s++) xv[m][s] = inside ? *reinterpret_cast<const f16x8 *>(x[m] + b * kBlockCols + 8 * s) : f16x8{};
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int f = 0; f < FT; f++) {
                const f16x8 wv = as_f16x8(mx_decode8(codes[f][s], scale[f]));
#pragma unroll
                for (int m = 0; m < MT; m++) acc[f][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wv, xv[m][s], acc[f][m], 0, 0, 0);
            }
    }
#pragma unroll
    for (int f = 0; f < FT; f++)
#pragma unroll
        for (int m = 0; m < MT; m++) red[((wave * FT + f) * MT + m) * kWave + lane] = acc[f][m];
    __syncthreads();
    if (wave >= FT * MT) return;
    f32x4 sum = red[wave * kWave + lane];
#pragma unroll
    for (int v = 1; v < kWaves4; v++) sum = sum + red[(v * FT * MT + wave) * kWave + lane];

    // sum[i] = C[row][feature n0 + i].
    const int row = m0 + 16 * (wave % MT) + c, n0 = 16 * (tile0 + wave / MT) + 4 * g;
    if (row >= M) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (n0 + i >= N) return;
        if constexpr (EP == EMBER_EPILOGUE_SILU_MUL) {
            if (i % 2 == 0)
                static_cast<f16 *>(C)[row * ldc + (n0 + i) / 2] = static_cast<f16>(clamp_half(silu(sum[i]) * sum[i + 1]));
        } else if constexpr (EP == EMBER_EPILOGUE_STORE_F16) {
            static_cast<f16 *>(C)[row * ldc + n0 + i] = static_cast<f16>(clamp_half(sum[i]));
        } else if constexpr (EP == EMBER_EPILOGUE_STORE_F32) {
            static_cast<float *>(C)[row * ldc + n0 + i] = sum[i];
        } else {
            static_cast<float *>(C)[row * ldc + n0 + i] += sum[i];
        }
    }
}

template <int EP>
hipError_t launch_gemv4_ep(const EmberGemv4Args &a, hipStream_t stream) {
    const f16 *A = static_cast<const f16 *>(a.A);
    const uint8_t *W = static_cast<const uint8_t *>(a.W);
    auto go = [&](auto kernel, int mt, int ft) {
        const dim3 grid(static_cast<unsigned>((a.N + 16 * ft - 1) / (16 * ft)), static_cast<unsigned>((a.M + 16 * mt - 1) / (16 * mt)));
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads4), 0, stream, A, a.lda, W, a.M, a.N, a.K, a.C, a.ldc);
    };
    if (a.M <= 16) go(gemv4_kernel<1, 1, EP>, 1, 1);
    else if (a.M <= 32) go(gemv4_kernel<2, 1, EP>, 2, 1);
    else go(gemv4_kernel<4, 1, EP>, 4, 1);
    return hipGetLastError();
}

// A thread per 8 columns (one word of codes).
__global__ void __launch_bounds__(256) gemv4_pack_kernel(const uint8_t *codes, const uint8_t *scales, int N, int K, uint8_t *out) {
    const int blocks = blocks_of(K);
    const int64_t words = static_cast<int64_t>((N + 15) / 16) * blocks * (kBlockCodes / 4);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < words; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int word = static_cast<int>(i % (kBlockCodes / 4)), lane = word / 4;
        const int64_t block = i / (kBlockCodes / 4);
        const int64_t row = block / blocks * 16 + lane % 16, col = block % blocks * kBlockCols + 32 * (lane / 16);
        const bool real = row < N && col < K;
        uint8_t *const dst = out + block * kBlockBytes;
        reinterpret_cast<uint32_t *>(dst)[word] = real ? reinterpret_cast<const uint32_t *>(codes + row * (K / 2) + col / 2)[word % 4] : 0u;
        if (word % 4 == 0) dst[kBlockCodes + lane] = real ? scales[row * (K / kMxGroup) + col / kMxGroup] : 0;
    }
}

// A thread per 8 columns, four lanes a group.
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

hipError_t launch_gemv4(const EmberGemv4Args &a, hipStream_t stream) {
    switch (a.epilogue) {
        case EMBER_EPILOGUE_STORE_F16: return launch_gemv4_ep<EMBER_EPILOGUE_STORE_F16>(a, stream);
        case EMBER_EPILOGUE_STORE_F32: return launch_gemv4_ep<EMBER_EPILOGUE_STORE_F32>(a, stream);
        case EMBER_EPILOGUE_ADD_F32: return launch_gemv4_ep<EMBER_EPILOGUE_ADD_F32>(a, stream);
        default: return launch_gemv4_ep<EMBER_EPILOGUE_SILU_MUL>(a, stream);
    }
}

}  // namespace ember::hip
