// Decode attention over a 4-bit K/V cache (kv4_layout.h).
//
// One wavefront per (sequence, query head): 64 tokens at a time, a lane
// computing the score of one token from its K words, then every lane the
// output channels of its share of the V words, with the online softmax's
// running maximum and sum.
#pragma once

#include "kv4_layout.h"
#include "paged_decode_kernels.h"

namespace xhip {

template <int KV> __device__ __forceinline__ float load_elem(const char *row, int i) {
    if constexpr (KV == KV_F16) return (float)((const _Float16 *)row)[i];
    else if constexpr (KV == KV_BF16)
        return __builtin_bit_cast(float, (uint32_t)((const uint16_t *)row)[i] << 16);
    else return ((const float *)row)[i];
}

template <int KV, int D>
__global__ __launch_bounds__(64) void paged_decode_kv4_kernel(const DecodeParams p) {
    constexpr int NG = kv4_groups(D);
    constexpr int DP = NG * kKv4Group;
    constexpr int EB = KvTraits<KV>::kBytes;
    constexpr int PAIRS = DP / 2;                  // channel pairs of a row
    constexpr int PER = (PAIRS + 63) / 64;         // of a lane
    __shared__ float s_q[DP], s_p[64];
    const int lane = threadIdx.x, head = blockIdx.x, s = blockIdx.y;
    const int kvh = head / p.group;
    const int L = seq_len_of(p, s);
    const int *bt = p.block_tables + (size_t)s * p.max_blocks;
    const char *q = q_row(p, s, head, D, EB);
    for (int i = lane; i < DP; i += 64) s_q[i] = i < D ? load_elem<KV>(q, i) : 0.0f;
    __syncthreads();
    const char *kb = (const char *)p.k + (size_t)kvh * (size_t)p.kv_head_stride;
    const char *vb = (const char *)p.v + (size_t)kvh * (size_t)p.kv_head_stride;
    float m = -INFINITY, l = 0.0f, o[PER][2] = {};
    auto tile_of = [&](const char *base, int t) -> const char * {
        const int blk = bt[t >> p.bs_shift];
        if (blk < 0) return nullptr;
        return base + (long long)blk * p.kv_block_stride +
               (size_t)((t & (p.block_size - 1)) / kKv4Tile) * kv4_tile_bytes(D);
    };
    for (int t0 = 0; t0 < L; t0 += 64) {
        const int t = t0 + lane;
        float sc = -INFINITY;
        if (const char *kt = t < L ? tile_of(kb, t) : nullptr) {
            sc = 0.0f;
            for (int g = 0; g < NG; g++) {
                float dot = 0.0f, sum = 0.0f;
                for (int qd = 0; qd < 4; qd++) {
                    const uint32_t w = *(const uint32_t *)(kt + kv4_k_word(NG, t & 15, qd, g));
                    for (int e = 0; e < 4; e++) {
                        const float q0 = s_q[32 * g + 8 * qd + 2 * e], q1 = s_q[32 * g + 8 * qd + 2 * e + 1];
                        dot += q0 * (float)(w >> (4 * e) & 15) + q1 * (float)(w >> (16 + 4 * e) & 15);
                        sum += q0 + q1;
                    }
                }
                sc += (float)*(const _Float16 *)(kt + kv4_step(NG, t & 15, g)) * dot +
                      (float)*(const _Float16 *)(kt + kv4_k_low(NG, t & 15, g)) * sum;
            }
            sc *= p.scale_log2;
        }
        const bool ok = t < L && bt[t >> p.bs_shift] >= 0;
        const float M = fmaxf(m, wave_max(sc));
        const float Ms = M == -INFINITY ? 0.0f : M;
        const float a = fast_exp2(m - Ms);
        const float e = ok ? fast_exp2(sc - Ms) : 0.0f;
        l = l * a + wave_sum(e);
        m = M;
        s_p[lane] = e;
        __syncthreads();
        for (int k = 0; k < PER; k++) o[k][0] *= a, o[k][1] *= a;
        for (int j = 0; j < 64 && t0 + j < L; j++) {
            const char *vt = tile_of(vb, t0 + j);
            if (!vt) continue;
            const int tt = (t0 + j) & 15;
            for (int k = 0; k < PER; k++) {
                const int pr = lane + 64 * k;
                if (pr >= PAIRS) continue;
                const int g = pr / 16, r = pr % 16;
                const uint32_t b = *(const uint8_t *)(vt + kv4_v_word(NG, tt >> 2, r, g) + kv4_v_byte(tt & 3));
                const float st = (float)*(const _Float16 *)(vt + kv4_step(NG, tt, g));
                const float lo = (float)*(const _Float16 *)(vt + kv4_v_low(NG, tt, g));
                o[k][0] += s_p[j] * fmaf(st, (float)(b & 15), lo);
                o[k][1] += s_p[j] * fmaf(st, (float)(b >> 4), lo);
            }
        }
        __syncthreads();
    }
    char *dst = o_row(p, s, head, D, EB);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    for (int k = 0; k < PER; k++)
        for (int e = 0; e < 2; e++) {
            const int c = 2 * (lane + 64 * k) + e;
            if (c < D) store_elem<KV>(dst, c, o[k][e] * inv);
        }
}

template <int KV>
static hipError_t launch_kv4_dtype(const DecodeParams &p, int head_size, hipStream_t st) {
    const dim3 grid((unsigned)p.num_heads, (unsigned)p.num_seqs);
    switch (head_size) {
#define XHIP_CASE(d) \
    case d: paged_decode_kv4_kernel<KV, d><<<grid, 64, 0, st>>>(p); return hipGetLastError();
        XHIP_CASE(32) XHIP_CASE(64) XHIP_CASE(80) XHIP_CASE(96) XHIP_CASE(112) XHIP_CASE(128)
        XHIP_CASE(192) XHIP_CASE(256)
#undef XHIP_CASE
    default: return hipErrorInvalidValue;
    }
}

}  // namespace xhip
