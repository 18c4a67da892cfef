// Fused QK-RMSNorm + rotate-half RoPE + write into 4-bit pages, gfx950.
//
// The arithmetic up to the codes is the f16 cache's append's in f32
// (kv_append.hip, same lanes: one wave per token and 8 heads, lane l serving
// head 8 * group + l / 8, elements 8 (l % 8) .. + 7 and those 64 further), so
// q_out has its bits and K and V are the values that f32 pages would hold. A
// lane's two pieces of 8 elements lie in one group of 32 each, whose largest
// magnitude four neighbouring lanes find by two quad permutations; a piece's
// codes are one 4-byte store.
//
// Bound by memory for many tokens, at 90% of a large copy's rate: us a launch,
// 9100 tokens of 32 + 8 + 8 heads 45 (4.3 TB/s), with k_out, v_out and a bias
// 62; 16,384 tokens of 16 + 8 + 8 heads 51; 32 tokens 4.4, a launch and three
// trips to memory. Waves without q or k heads take no sine and cosine, waves
// without heads end at once (56, 68 and 59 us before). Tried: a wave for all
// heads of a token, one sine and cosine for them all (8.0 us for 32 tokens, 55
// for 9100: 112 registers leave half the waves); sines and cosines once for 2 or
// 4 tokens' waves, through LDS (53 and 63 for 9100).
#include "device.hpp"
#include "four_bit.hpp"
#include "kernels.hpp"

namespace ember::hip {
namespace {

constexpr int kWavesPerBlock = 4;
constexpr int kLanesPerHead = 8;
constexpr int kHeadsPerWave = kWave / kLanesPerHead;
constexpr int kElems = kHeadDim / 2 / kLanesPerHead;  // elements per lane in each half

__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, dpp_mov<kDppQuadXor1>(x));
    return fmaxf(x, dpp_mov<kDppQuadXor2>(x));
}

__device__ __forceinline__ float largest(const float (&x)[kElems]) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < kElems; e++) m = fmaxf(m, fabsf(x[e]));
    return quad_max(m);
}

__global__ void __launch_bounds__(kWavesPerBlock * kWave)
    kv4_append_kernel(const int32_t *positions, const int32_t *token_seq, const float *inv_freq, const void *qkv,
                      const int32_t *block_tables, int n_heads, int n_kv, int max_blocks, EmberKv4AppendArgs a) {
    constexpr int D = kHeadDim, HALF = D / 2;
    const int t = blockIdx.x;
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    const int group = static_cast<int>(blockIdx.y) * kWavesPerBlock + uniform(static_cast<int>(threadIdx.x) / kWave);
    const int total = n_heads + 2 * n_kv;
    if (group * kHeadsPerWave >= total) return;
    const bool turns = group * kHeadsPerWave < n_heads + n_kv;  // some of the wave's heads are q or k
    const int head = group * kHeadsPerWave + lane / kLanesPerHead;
    const int piece = lane % kLanesPerHead, e0 = piece * kElems;
    const bool live = head < total;

    // Loads in the order that their results are needed: the frequency, the token's position and row, the head's elements,
    // then the block id, which needs the first two (clamped into the tables; a token outside them stores no page).
    const float freq = inv_freq[lane];
    __builtin_amdgcn_sched_barrier(0);
    const int pos = positions[t];
    const int seq = token_seq[t];
    const f16 *src = static_cast<const f16 *>(qkv) + (static_cast<int64_t>(t) * total + min(head, total - 1)) * D;
    const f16x8 r0 = *reinterpret_cast<const f16x8 *>(src + e0), r1 = *reinterpret_cast<const f16x8 *>(src + HALF + e0);
    __builtin_amdgcn_sched_barrier(0);
    const bool is_q = head < n_heads, is_k = !is_q && head < n_heads + n_kv;
    const int page = pos / kPage;
    const bool slot_ok = pos >= 0 && page < max_blocks && seq >= 0 && seq < a.rows;
    const int block = block_tables[static_cast<int64_t>(min(max(seq, 0), a.rows - 1)) * max_blocks + min(max(page, 0), max_blocks - 1)];

    float sn[kElems], cs[kElems];
    if (turns) {
        const float angle = static_cast<float>(pos) * freq;
        double sd, cd;
        sincos(static_cast<double>(angle), &sd, &cd);
        const float s_f = static_cast<float>(sd), c_f = static_cast<float>(cd);
#pragma unroll
        for (int e = 0; e < kElems; e++) sn[e] = __shfl(s_f, e0 + e, kWave), cs[e] = __shfl(c_f, e0 + e, kWave);
    }

    float x0[kElems], x1[kElems];
#pragma unroll
    for (int e = 0; e < kElems; e++) x0[e] = static_cast<float>(r0[e]), x1[e] = static_cast<float>(r1[e]);
    if (a.bias) {
        const float *b = a.bias + min(head, total - 1) * D;
#pragma unroll
        for (int e = 0; e < kElems; e++) x0[e] = x0[e] + b[e0 + e], x1[e] = x1[e] + b[HALF + e0 + e];
    }

    double ss[kElems] = {};
    if (turns && a.q_norm) {
        // Sum of squares over the head in double, in kv_append.hip's pairing order.
#pragma unroll
        for (int e = 0; e < kElems; e++)
            ss[e] = static_cast<double>(x0[e]) * x0[e] + static_cast<double>(x1[e]) * x1[e];
#pragma unroll
        for (int o = kLanesPerHead / 2; o > 0; o >>= 1) {
#pragma unroll
            for (int e = 0; e < kElems; e++) ss[e] += __shfl_xor(ss[e], o, kLanesPerHead);
        }
#pragma unroll
        for (int o = kElems / 2; o > 0; o >>= 1) {
#pragma unroll
            for (int e = 0; e < o; e++) ss[e] += ss[e + o];
        }
    }

    if (is_q || is_k) {
        const float *w = is_q ? a.q_norm : a.k_norm;
        if (w) {
            const float scale = static_cast<float>(1.0 / sqrt(ss[0] / kHeadDim + static_cast<double>(a.eps)));
#pragma unroll
            for (int e = 0; e < kElems; e++) {
                x0[e] = w[e0 + e] * (x0[e] * scale);
                x1[e] = w[HALF + e0 + e] * (x1[e] * scale);
            }
        }
#pragma unroll
        for (int e = 0; e < kElems; e++) {
            const float lo = x0[e], hi = x1[e];
            x0[e] = lo * cs[e] - hi * sn[e];
            x1[e] = hi * cs[e] + lo * sn[e];
        }
    }
    if (!live) return;

    if (is_q) {
        f16 *dst = static_cast<f16 *>(a.q_out) + (static_cast<int64_t>(t) * n_heads + head) * D;
        f16x8 v0, v1;
#pragma unroll
        for (int e = 0; e < kElems; e++) v0[e] = static_cast<f16>(x0[e]), v1[e] = static_cast<f16>(x1[e]);
        *reinterpret_cast<f16x8 *>(dst + e0) = v0;
        *reinterpret_cast<f16x8 *>(dst + HALF + e0) = v1;
        return;
    }
#pragma unroll
    for (int e = 0; e < kElems; e++) x0[e] = clamp_half(x0[e]), x1[e] = clamp_half(x1[e]);
    const int b0 = mx_scale_byte(largest(x0)), b1 = mx_scale_byte(largest(x1));
    const float s0 = mx_scale(b0), s1 = mx_scale(b1);
    const uint32_t w0 = mx_encode8(x0, s0), w1 = mx_encode8(x1, s1);
    const int kvh = is_k ? head - n_heads : head - n_heads - n_kv;
    if (a.k_out) {
        f16 *dst = static_cast<f16 *>(is_k ? a.k_out : a.v_out) + (static_cast<int64_t>(t) * n_kv + kvh) * D;
        *reinterpret_cast<u32x4 *>(dst + e0) = mx_decode8(w0, s0);
        *reinterpret_cast<u32x4 *>(dst + HALF + e0) = mx_decode8(w1, s1);
    }
    if (!slot_ok || block < 0 || block >= a.num_blocks) return;  // never write outside the pool
    uint8_t *dst = static_cast<uint8_t *>(a.pool) + (static_cast<int64_t>(block) * n_kv + kvh) * kKv4Page;
    const int slot = pos % kPage, quad = piece / 4;  // the pieces are in groups `quad` and quad + 2
    if (is_k) {
        uint8_t *const codes = dst + slot * (D / 2) + 4 * piece;
        *reinterpret_cast<uint32_t *>(codes) = w0;
        *reinterpret_cast<uint32_t *>(codes + D / 4) = w1;
        if (piece % 4 == 0) {
            dst[kKv4KeyScales + 4 * slot + quad] = static_cast<uint8_t>(b0);
            dst[kKv4KeyScales + 4 * slot + quad + 2] = static_cast<uint8_t>(b1);
        }
    } else {
        uint8_t *const codes = dst + kKv4Values + 256 * (slot / 4) + 4 * (slot % 4) + 16 * piece;
        *reinterpret_cast<uint32_t *>(codes) = w0;
        *reinterpret_cast<uint32_t *>(codes + 128) = w1;
        if (piece % 4 == 0) {
            dst[kKv4ValueScales + kPage * quad + slot] = static_cast<uint8_t>(b0);
            dst[kKv4ValueScales + kPage * (quad + 2) + slot] = static_cast<uint8_t>(b1);
        }
    }
}

}  // namespace

hipError_t launch_kv4_append(const EmberKv4AppendArgs &a, hipStream_t stream) {
    const int groups = (a.n_heads + 2 * a.n_kv + kHeadsPerWave - 1) / kHeadsPerWave;
    const dim3 grid(static_cast<unsigned>(a.T), static_cast<unsigned>((groups + kWavesPerBlock - 1) / kWavesPerBlock));
    hipLaunchKernelGGL(kv4_append_kernel, grid, dim3(kWavesPerBlock * kWave), 0, stream, a.positions, a.token_seq, a.inv_freq,
                       a.qkv, a.block_tables, a.n_heads, a.n_kv, a.max_blocks, a);
    return hipGetLastError();
}

}  // namespace ember::hip
