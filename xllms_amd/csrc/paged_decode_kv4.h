// Decode attention over a 4-bit K/V cache (kv4_layout.h), on the matrix cores.
//
// The work split (stream-K over the batch) and the merge are the fp16 path's
// (paged_decode_params.h, paged_decode_kernels.h, next_piece of
// paged_decode_mfma.h), with tiles of 32 tokens: two 16-token cache tiles a and
// b, which may lie in different pages.  One wavefront serves R blocks of 16
// query heads of one kv head.  With j = lane % 16 and quarter q = lane / 16:
//
//   scores  S[t][h] = sum_g step[t][g] * (sum_{c in g} code[t][c] q[h][c])
//                     + sum_g low[t][g] * (sum_{c in g} q[h][c])
//     One v_mfma_f32_16x16x32_f16 per group and cache tile, A = 16 tokens' codes
//     of the group's 32 channels (lane: token j, channels 32g + 8q..+7, one word),
//     B = the queries of 16 heads (lane: head j, the same channels).  A code
//     masked out of its word is an fp16 number by itself, code * 2^-24 (a
//     subnormal; the matrix cores keep them) or, from bits 4-7, code * 2^-20,
//     for which the query of that channel carries 1/16.  The lane holds the
//     sums of tokens 4q..4q+3 of head j and applies the steps in fp32.  The
//     second sum is one more MFMA over the groups: A = lows (lane: token j),
//     B = the groups' query sums, as two fp16 parts.
//     Queries are scaled by a power of two per head so that the largest lies in
//     [2^14, 2^15): any finite magnitude of any type fits fp16.  An fp32 query
//     is two fp16 parts (22 bits).
//   softmax per head j over the lane's 8 scores; the maximum goes across the
//     four quarters, and the outputs are rescaled, only when a score passes the
//     running maximum (past the first few hundred tokens most tiles pass by).
//   PV      O[c][h] = sum_t (p[t][h] step[t][g]) code[t][c] + sum_t p[t][h] low[t][g]
//     B = p * step for the group's two channel blocks (lane: head j, its own 8
//     tokens: exactly where the softmax left them), A = codes (lane: channel
//     pair j, 4 tokens of a and 4 of b; the even channel from the low nibbles,
//     the odd one, 16 times as large, from the high ones).  Row i of a block is
//     channel 32g + 2i (+ 1), so a lane ends with 8 neighbouring channels of
//     each group.  The second sum is one more MFMA, A = lows (lane: group j).
//     Weights are scaled by 2^13, which
//     keeps p * step clear of fp16's subnormals: at 2^13 a step of up to 2
//     (values that span 30) leaves p * step below 2^14.  A tile with a larger
//     step is summed on its own with p * step / 2^12 and added back times 2^12.
//     p * step and p go in as two fp16 parts, hi + lo (22 bits); for a bf16
//     output, whose half step is 2^-8, as one (half step 2^-11).
//
// Per 32 tokens of a kv head at head_size 128 that is 5120 bytes, and about 230
// vector instructions and 28-52 MFMAs: the unpacking is 5 instructions per 8
// codes.
#pragma once

#include "kv4_layout.h"
#include "paged_decode_dispatch.h"
#include "paged_decode_mfma.h"

namespace xhip {

constexpr int kKv4TileTokens = 32;  // tokens of a tile: two cache tiles
constexpr int kKv4Waves = kMfmaWavesPerGroup;

template <int D> struct Kv4Geometry {
    static constexpr int NG = kv4_groups(D);
    static constexpr int kBytes = kv4_tile_bytes(D);
    static constexpr int kLowWords = (NG + 1) / 2;  // a token's lows of K
};

// One lane's share of a cache tile.
template <int D> struct Kv4Keys {
    uint32_t code[Kv4Geometry<D>::NG];      // token j, quarter q of each group
    u32x2 step[Kv4Geometry<D>::NG];         // tokens 4q..4q+3
    uint32_t low[Kv4Geometry<D>::kLowWords];  // token j
};
template <int D> struct Kv4Values {
    uint32_t code[Kv4Geometry<D>::NG];  // tokens 4q..4q+3, channel pair j of each group
    u32x2 step[Kv4Geometry<D>::NG];     // tokens 4q..4q+3
    u32x2 low;                          // tokens 4q..4q+3 of group j (past the groups: the last)
};

template <int N>
__device__ __forceinline__ void buf_words(__amdgpu_buffer_rsrc_t r, int off, uint32_t (&w)[N]) {
    if constexpr (N >= 4) {
        const u32x4 x = buf_load<4, kStreamPolicy>(r, (uint32_t)off);
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = lane_word(x, i);
        if constexpr (N > 4) {
            uint32_t rest[N - 4];
            buf_words<N - 4>(r, off + 16, rest);
#pragma unroll
            for (int i = 4; i < N; i++) w[i] = rest[i - 4];
        }
    } else {
        const u32x4 x = buf_load<N, kStreamPolicy>(r, (uint32_t)off);
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = lane_word(x, i);
    }
}

template <int NG>
__device__ __forceinline__ void buf_pairs(__amdgpu_buffer_rsrc_t r, int off, u32x2 (&v)[NG]) {
    uint32_t w[2 * NG];
    buf_words<2 * NG>(r, off, w);
#pragma unroll
    for (int g = 0; g < NG; g++) v[g] = u32x2{w[2 * g], w[2 * g + 1]};
}

// Buffer over one cache tile; with ok false every load from it is zero and
// touches no memory.
template <int D> __device__ __forceinline__ __amdgpu_buffer_rsrc_t kv4_rsrc(const char *tile, bool ok) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)tile, (short)0,
                                             ok ? Kv4Geometry<D>::kBytes : 0, 0x00020000);
}

template <int D>
__device__ __forceinline__ void kv4_load_keys(__amdgpu_buffer_rsrc_t r, int lane, Kv4Keys<D> &k) {
    constexpr int NG = Kv4Geometry<D>::NG;
    const int j = lane & 15, q = lane >> 4;
    buf_words<NG>(r, kv4_k_word(NG, j, q, 0), k.code);
    buf_pairs<NG>(r, kv4_step(NG, 4 * q, 0), k.step);
    if constexpr (NG == 1) {
        k.low[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, kv4_k_low(NG, j, 0), 0, kStreamPolicy);
    } else if constexpr (NG == 3) {
        uint32_t w[1];
        buf_words<1>(r, kv4_k_low(NG, j, 0), w);
        k.low[0] = w[0];
        k.low[1] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, kv4_k_low(NG, j, 2), 0, kStreamPolicy);
    } else {
        buf_words<NG / 2>(r, kv4_k_low(NG, j, 0), k.low);
    }
}

template <int D>
__device__ __forceinline__ void kv4_load_values(__amdgpu_buffer_rsrc_t r, int lane, Kv4Values<D> &v) {
    constexpr int NG = Kv4Geometry<D>::NG;
    const int j = lane & 15, q = lane >> 4;
    buf_words<NG>(r, kv4_v_word(NG, q, j, 0), v.code);
    buf_pairs<NG>(r, kv4_step(NG, 4 * q, 0), v.step);
    uint32_t w[2];
    buf_words<2>(r, kv4_v_low(NG, 4 * q, j < NG ? j : NG - 1), w);
    v.low = u32x2{w[0], w[1]};
}

__device__ __forceinline__ f32x4 mfma_h(u32x4 a, u32x4 b, f32x4 c) {
    return mfma_qk<KV_F16>(a, b, c);
}

__device__ __forceinline__ uint32_t half_pair(float a, float b) { return pack16<KV_F16>(a, b); }

// Two codes of a word as fp16: nibbles 0 and 4 (times 2^-24), or with HIGH
// nibbles 1 and 5 (times 2^-20).
template <bool HIGH> __device__ __forceinline__ uint32_t code_pair(uint32_t w) {
    return w & (HIGH ? 0x00f000f0u : 0x000f000fu);
}

// Query operands of one head block.  kTerms: fp16 parts of a query element.
template <int KV, int D> struct Kv4Query {
    static constexpr int kTerms = KV == KV_F32 ? 2 : 1;
    u32x4 q[kTerms][Kv4Geometry<D>::NG];
    u32x4 sums;        // the groups' sums: quarter q's 4 groups, hi and lo
    float a, b;        // score (log2 units) = a * (code part) + b * (low part)
};

template <int KV, int D>
__device__ __forceinline__ void kv4_load_query(const DecodeParams &p, const MfmaPiece &pc, int lane,
                                               int head0, int heads, Kv4Query<KV, D> &o) {
    using G = Kv4Geometry<D>;
    constexpr int NG = G::NG, EB = KvTraits<KV>::kBytes;
    const int j = lane & 15, q = lane >> 4;
    float x[NG][8];
    float top = 0.0f;
    bool finite = true;
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const int c = 32 * g + 8 * q;
        if (j < heads && (D % 32 == 0 || c < D)) {
            const char *src = q_row(p, pc.s, pc.kvh * p.group + head0 + j, D, EB) + (size_t)c * EB;
            if constexpr (KV == KV_F32) {
                chunk_to_float<KV_F32, 4>(load16(src), *(float(*)[4]) & x[g][0]);
                chunk_to_float<KV_F32, 4>(load16(src + 16), *(float(*)[4]) & x[g][4]);
            } else {
                chunk_to_float<KV, 8>(load16(src), x[g]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[g][e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            top = fmaxf(top, fabsf(x[g][e]));
            finite &= fabsf(x[g][e]) < INFINITY;
        }
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    // every quarter of the head
    const unsigned long long bad = __ballot(!finite);
    const bool row_bad = ((bad | bad >> 16 | bad >> 32 | bad >> 48) >> j & 1) != 0;
    const int ex = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
    float sum[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[g][e] = __builtin_amdgcn_ldexpf(x[g][e], 15 - ex);
            s += x[g][e];
            if (e & 2) x[g][e] *= 0.0625f;  // its codes come 16 times as large
        }
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        sum[g] = s * (1.0f / 512.0f);  // below 2^11
        u32x4 hi;
#pragma unroll
        for (int e = 0; e < 4; e++) hi[e] = half_pair(x[g][2 * e], x[g][2 * e + 1]);
        o.q[0][g] = hi;
        if constexpr (KV == KV_F32) {
            u32x4 lo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const f32x2 r = unpack16<KV_F16>(lane_word(hi, e));
                lo[e] = half_pair(x[g][2 * e] - r.x, x[g][2 * e + 1] - r.y);
            }
            o.q[1][g] = lo;
        }
    }
    // Quarter q < 2 holds groups 4q..4q+3; the other quarters nothing.  A query
    // with an infinity or NaN makes every score of its head NaN.
    float s4[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float s0 = i < NG ? sum[i < NG ? i : 0] : 0.0f;
        const float s1 = 4 + i < NG ? sum[4 + i < NG ? 4 + i : 0] : 0.0f;
        s4[i] = q == 0 ? s0 : q == 1 ? s1 : 0.0f;
    }
    if (row_bad && q == 0) s4[0] = __builtin_nanf("");
    const uint32_t h01 = half_pair(s4[0], s4[1]), h23 = half_pair(s4[2], s4[3]);
    const f32x2 r01 = unpack16<KV_F16>(h01), r23 = unpack16<KV_F16>(h23);
    o.sums = u32x4{h01, h23, half_pair(s4[0] - r01.x, s4[1] - r01.y),
                   half_pair(s4[2] - r23.x, s4[3] - r23.y)};
    o.a = __builtin_amdgcn_ldexpf(p.scale_log2, ex - 15 + 24);
    o.b = __builtin_amdgcn_ldexpf(p.scale_log2, ex - 15 + 9);
}

// Running state of one head block: lane (q, j) owns head j.
template <int D> struct Kv4State {
    f32x4 o[Kv4Geometry<D>::NG][2];  // [group][odd channel], rows 4q..4q+3: 2^-24 and 2^-20 of it
    f32x4 low;                       // row 4q + i: group 4q + i's sum of p * low
    float l;                         // this lane's part of the running sum
    float base;                      // weights of head j are 2^(score - base)
    float limit;                     // score - base up to which they are kept: 13; -inf
                                     // (and base 0) before the head's first score
};

constexpr float kKv4Top = 13.0f;  // log2 of the largest weight

// Scores of one cache tile against one head block, less `base` (log2 units):
// tokens 4q..4q+3 of head j.
template <int KV, int D>
__device__ __forceinline__ void kv4_scores(const Kv4Keys<D> &k, const Kv4Query<KV, D> &qr, int lane,
                                           float base, float (&x)[4]) {
    using G = Kv4Geometry<D>;
    constexpr int NG = G::NG;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 a;  // lows of this lane's quarter's groups, twice (the sums' hi and lo)
    {
        uint32_t w0 = k.low[0], w1 = G::kLowWords > 1 ? k.low[G::kLowWords > 1 ? 1 : 0] : 0u;
        if constexpr (NG > 4) {
            const bool up = (lane >> 4) == 1;
            w0 = up ? k.low[2] : w0;
            w1 = up ? (G::kLowWords > 3 ? k.low[G::kLowWords > 3 ? 3 : 0] : 0u) : w1;
        }
        a = u32x4{w0, w1, w0, w1};
    }
    const f32x4 lows = mfma_h(a, qr.sums, zero);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const uint32_t w = k.code[g], y = w >> 8;
        const u32x4 c = {code_pair<false>(w), code_pair<true>(w), code_pair<false>(y), code_pair<true>(y)};
        f32x4 t = mfma_h(c, qr.q[0][g], zero);
        if constexpr (KV == KV_F32) t = mfma_h(c, qr.q[1][g], t);
        const f16x2 s01 = __builtin_bit_cast(f16x2, (uint32_t)k.step[g].x);
        const f16x2 s23 = __builtin_bit_cast(f16x2, (uint32_t)k.step[g].y);
        s[0] = fmaf((float)s01.x, t[0], s[0]);
        s[1] = fmaf((float)s01.y, t[1], s[1]);
        s[2] = fmaf((float)s23.x, t[2], s[2]);
        s[3] = fmaf((float)s23.y, t[3], s[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = fmaf(qr.a, s[i], fmaf(qr.b, lows[i], -base));
}

// O += P V of one tile and head block.  pe: the weights of the lane's tokens
// 4q..4q+3 of a, then of b.  BIG: a step of the tile is 2 or more.
template <int KV, int D, bool BIG>
__device__ __forceinline__ void kv4_pv(const Kv4Values<D> &va, const Kv4Values<D> &vb,
                                       const float (&pe)[8], Kv4State<D> &st) {
    constexpr int NG = Kv4Geometry<D>::NG;
    constexpr bool kLo = KV != KV_BF16;  // a second fp16 part of the weights
    constexpr float kDown = BIG ? 1.0f / 4096.0f : 1.0f;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    {
        u32x4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            hi[i] = half_pair(pe[2 * i], pe[2 * i + 1]);
            if constexpr (kLo) {
                const f32x2 r = unpack16<KV_F16>(lane_word(hi, i));
                lo[i] = half_pair(pe[2 * i] - r.x, pe[2 * i + 1] - r.y);
            }
        }
        const u32x4 a = {va.low.x, va.low.y, vb.low.x, vb.low.y};
        st.low = mfma_h(a, hi, st.low);
        if constexpr (kLo) st.low = mfma_h(a, lo, st.low);
    }
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const uint32_t sw[4] = {va.step[g].x, va.step[g].y, vb.step[g].x, vb.step[g].y};
        f16x8 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f16x2 s = __builtin_bit_cast(f16x2, sw[i]);
            const float w0 = BIG ? pe[2 * i] * kDown : pe[2 * i];
            const float w1 = BIG ? pe[2 * i + 1] * kDown : pe[2 * i + 1];
            const _Float16 h0 = (_Float16)(w0 * (float)s.x), h1 = (_Float16)(w1 * (float)s.y);
            hi[2 * i] = h0;
            hi[2 * i + 1] = h1;
            if constexpr (kLo) {
                lo[2 * i] = (_Float16)fmaf(w0, (float)s.x, -(float)h0);
                lo[2 * i + 1] = (_Float16)fmaf(w1, (float)s.y, -(float)h1);
            }
        }
        const u32x4 ph = __builtin_bit_cast(u32x4, hi), pl = __builtin_bit_cast(u32x4, lo);
        const uint32_t x = va.code[g], x8 = x >> 8, y = vb.code[g], y8 = y >> 8;
        const u32x4 even = {code_pair<false>(x), code_pair<false>(x8), code_pair<false>(y), code_pair<false>(y8)};
        const u32x4 odd = {code_pair<true>(x), code_pair<true>(x8), code_pair<true>(y), code_pair<true>(y8)};
        f32x4 t0 = mfma_h(even, ph, BIG ? zero : st.o[g][0]);
        f32x4 t1 = mfma_h(odd, ph, BIG ? zero : st.o[g][1]);
        if constexpr (kLo) {
            t0 = mfma_h(even, pl, t0);
            t1 = mfma_h(odd, pl, t1);
        }
        st.o[g][0] = BIG ? st.o[g][0] + t0 * 4096.0f : t0;
        st.o[g][1] = BIG ? st.o[g][1] + t1 * 4096.0f : t1;
    }
}

// The state's value of the lane's 8 channels of group g (32g + 8q..+7), not
// yet divided by l.
template <int D>
__device__ __forceinline__ void kv4_channels(const Kv4State<D> &st, int g, int lane, float (&f)[8]) {
    // the group's low sum, from its quarter
    const float own = st.low[g & 3];
    const float low = __shfl(own, (g >> 2) * 16 + (lane & 15));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f[2 * i] = fmaf(st.o[g][0][i], 16777216.0f, low);
        f[2 * i + 1] = fmaf(st.o[g][1][i], 1048576.0f, low);
    }
}

// A finished piece: its output rows, or its fp32 partial in the piece's slot.
template <int KV, int D, int R>
__device__ __forceinline__ void kv4_write(const DecodeParams &p, const MfmaPiece &pc, int lane,
                                          const Kv4State<D> (&st)[R]) {
    constexpr int GT = kMfmaHeads * R, EB = KvTraits<KV>::kBytes, NG = Kv4Geometry<D>::NG;
    const int j = lane & 15, q = lane >> 4;
    const int g0 = pc.ht * GT;
    const int nh = min(GT, p.group - g0);
#pragma unroll
    for (int b = 0; b < R; b++) {
        float l = st[b].l;
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const int hj = 16 * b + j;
        const float mul = !pc.whole ? 1.0f : l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const size_t row = ((size_t)pc.slot * GT + hj) * D;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float f[8];
            kv4_channels<D>(st[b], g, lane, f);
            const int c = 32 * g + 8 * q;
            if (hj >= nh || (D % 32 != 0 && c >= D)) continue;
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] *= mul;
            if (pc.whole)
                store_elems<KV>(o_row(p, pc.s, pc.kvh * p.group + g0 + hj, D, EB), c, f);
            else
                store_floats(p.ws_o + row + c, f);
        }
        if (!pc.whole && hj < nh && q == 0) {
            float *ml = p.ws_ml + ((size_t)pc.slot * GT + hj) * 2;
            ml[0] = st[b].limit == -INFINITY ? -INFINITY : st[b].base;
            ml[1] = l;
        }
    }
}

// Where a tile's two cache tiles are: page ids (negative: not there) and the
// first token.
struct Kv4TileRef {
    int t0, t_end, blk_a, blk_b;
};

template <int D>
__device__ __forceinline__ const char *kv4_tile_at(const DecodeParams &p, const char *base, int t, int blk) {
    return base + (long long)blk * p.kv_block_stride +
           (long long)((t & (p.block_size - 1)) / kKv4Tile) * Kv4Geometry<D>::kBytes;
}

template <int D>
__device__ __forceinline__ void kv4_load_k(const DecodeParams &p, const char *kb, const Kv4TileRef &r,
                                           int lane, Kv4Keys<D> (&k)[2]) {
    kv4_load_keys<D>(kv4_rsrc<D>(kv4_tile_at<D>(p, kb, r.t0, r.blk_a), r.blk_a >= 0), lane, k[0]);
    kv4_load_keys<D>(kv4_rsrc<D>(kv4_tile_at<D>(p, kb, r.t0 + 16, r.blk_b), r.blk_b >= 0), lane, k[1]);
}

template <int D>
__device__ __forceinline__ void kv4_load_v(const DecodeParams &p, const char *vb, const Kv4TileRef &r,
                                           int lane, Kv4Values<D> (&v)[2]) {
    kv4_load_values<D>(kv4_rsrc<D>(kv4_tile_at<D>(p, vb, r.t0, r.blk_a), r.blk_a >= 0), lane, v[0]);
    kv4_load_values<D>(kv4_rsrc<D>(kv4_tile_at<D>(p, vb, r.t0 + 16, r.blk_b), r.blk_b >= 0), lane, v[1]);
}

// Page ids of the piece's cache tiles first .. first + 63, lane i holding
// cache tile first + i (past the piece's end: -1).
__device__ __forceinline__ int kv4_load_ids(const DecodeParams &p, const int *__restrict__ tables,
                                            const MfmaPiece &pc, int first, int lane) {
    const int *bt = tables + (size_t)pc.s * p.max_blocks;
    const int t = pc.t_begin + kKv4Tile * (first + lane);
    const int id = bt[(t < pc.t_end ? t : pc.t_end - 1) >> p.bs_shift];
    return t < pc.t_end ? id : -1;
}

// Wavefronts per SIMD the kernel is compiled for.
constexpr int kv4_waves_per_simd(int head_size, int row_blocks) {
    return head_size > 128 || row_blocks > 1 ? (head_size * row_blocks > 256 ? 1 : 2) : 2;
}

template <int KV, int D, int R>
__global__ __launch_bounds__(64 * kKv4Waves, (kv4_waves_per_simd(D, R))) void paged_decode_partition_kv4_kernel(
    const DecodeParams p, const int *__restrict__ lens, const int *__restrict__ tables) {
    extern __shared__ int pre[];  // num_seqs + 1 split-unit prefixes
    constexpr int TT = kKv4TileTokens;
    batch_prefix<TT, kKv4Waves>(p, pre);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int total = pre[p.num_seqs];
    const int w = logical_block(p, total) * kKv4Waves + wave;
    const int tpw = tiles_per_wave(total, p.num_waves, p.min_tiles_per_wave);
    if (blockIdx.x == 0 && threadIdx.x == 0) p.ws_prefix[p.num_seqs + 1] = tpw;  // for the merge
    const long long g_lo = (long long)w * tpw;
    if (g_lo >= total) return;
    RangeCursor cur;
    cur.g = (int)g_lo;
    cur.g_end = min(total, cur.g + tpw);
    cur.first = 1;
    cur.w = w;
    cur.ht = -1;
    {
        int lo = 0, hi = p.num_seqs - 1;  // the sequence holding unit g
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= cur.g) lo = mid; else hi = mid - 1;
        }
        cur.s = __builtin_amdgcn_readfirstlane(lo);
    }
    MfmaPiece pc;
    if (!next_piece<TT>(p, lens, pre, cur, pc)) return;
    int ids = kv4_load_ids(p, tables, pc, 0, lane);
    Kv4Keys<D> k[2];
    Kv4Values<D> v[2];
    Kv4TileRef at = {pc.t_begin, pc.t_end, __builtin_amdgcn_readlane(ids, 0), __builtin_amdgcn_readlane(ids, 1)};
    kv4_load_k<D>(p, (const char *)p.k + (size_t)pc.kvh * p.kv_head_stride, at, lane, k);
    kv4_load_v<D>(p, (const char *)p.v + (size_t)pc.kvh * p.kv_head_stride, at, lane, v);
    while (true) {
        Kv4Query<KV, D> qr[R];
        Kv4State<D> st[R];
        const int g0 = pc.ht * kMfmaHeads * R;
#pragma unroll
        for (int b = 0; b < R; b++) {
            kv4_load_query<KV, D>(p, pc, lane, g0 + 16 * b, p.group - g0 - 16 * b, qr[b]);
#pragma unroll
            for (int g = 0; g < Kv4Geometry<D>::NG; g++)
                st[b].o[g][0] = st[b].o[g][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            st[b].low = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            st[b].l = st[b].base = 0.0f;
            st[b].limit = -INFINITY;
        }
        MfmaPiece pn = pc;
        const bool has_next = next_piece<TT>(p, lens, pre, cur, pn);
        const int ids_n = kv4_load_ids(p, tables, pn, 0, lane);
        const int ntiles = (pc.t_end - pc.t_begin + TT - 1) / TT;
        for (int i = 0; i < ntiles; i++) {
            // the next tile: this piece's, the next piece's first, or none
            Kv4TileRef nx;
            const bool in_piece = i + 1 < ntiles;
            if (in_piece) {
                const int n = 2 * (i + 1) & 63;
                if (n == 0) ids = kv4_load_ids(p, tables, pc, 2 * (i + 1), lane);
                nx = {at.t0 + TT, pc.t_end, __builtin_amdgcn_readlane(ids, n), __builtin_amdgcn_readlane(ids, n + 1)};
            } else if (has_next) {
                nx = {pn.t_begin, pn.t_end, __builtin_amdgcn_readlane(ids_n, 0), __builtin_amdgcn_readlane(ids_n, 1)};
            } else {
                nx = {0, 0, -1, -1};
            }
            const int kvh_n = in_piece ? pc.kvh : pn.kvh;

            float x[R][8];
#pragma unroll
            for (int b = 0; b < R; b++) {
                kv4_scores<KV, D>(k[0], qr[b], lane, st[b].base, *(float(*)[4]) & x[b][0]);
                kv4_scores<KV, D>(k[1], qr[b], lane, st[b].base, *(float(*)[4]) & x[b][4]);
            }
            kv4_load_k<D>(p, (const char *)p.k + (size_t)kvh_n * p.kv_head_stride, nx, lane, k);

            const int q4 = (lane >> 4) * 4;
            const bool full = at.t0 + TT <= at.t_end && at.blk_a >= 0 && at.blk_b >= 0;
            if (!full) {
                // tokens past the end or in missing pages: no weight, and no
                // step or low of theirs (whatever the slots hold) in a product
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    bool ok[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        ok[e] = (h ? at.blk_b : at.blk_a) >= 0 && at.t0 + 16 * h + q4 + e < at.t_end;
#pragma unroll
                        for (int b = 0; b < R; b++) x[b][4 * h + e] = ok[e] ? x[b][4 * h + e] : -INFINITY;
                    }
                    const uint32_t m01 = (ok[0] ? 0xFFFFu : 0u) | (ok[1] ? 0xFFFF0000u : 0u);
                    const uint32_t m23 = (ok[2] ? 0xFFFFu : 0u) | (ok[3] ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int g = 0; g < Kv4Geometry<D>::NG; g++) {
                        v[h].step[g].x &= m01;
                        v[h].step[g].y &= m23;
                    }
                    v[h].low.x &= m01;
                    v[h].low.y &= m23;
                }
            }
            uint32_t steps = 0;
#pragma unroll
            for (int g = 0; g < Kv4Geometry<D>::NG; g++)
                steps |= v[0].step[g].x | v[0].step[g].y | v[1].step[g].x | v[1].step[g].y;
            const bool big = __any((steps & 0x40004000u) != 0);  // fp16: 2 or more
#pragma unroll
            for (int b = 0; b < R; b++) {
                Kv4State<D> &s = st[b];
                float mx = x[b][0];
#pragma unroll
                for (int e = 1; e < 8; e++) mx = fmaxf(mx, x[b][e]);
                if (__any(mx > s.limit)) {
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    const bool up = mx > s.limit;
                    const float base = up ? s.base + (mx - kKv4Top) : s.base;
                    const float alpha = up && s.limit != -INFINITY ? fast_exp2(s.base - base) : 1.0f;
                    s.base = base;
                    s.limit = up ? kKv4Top : s.limit;
                    s.l *= alpha;
                    s.low *= alpha;
#pragma unroll
                    for (int g = 0; g < Kv4Geometry<D>::NG; g++) {
                        s.o[g][0] *= alpha;
                        s.o[g][1] *= alpha;
                    }
                    // (the largest weight is 2^13 to the bit)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[b][e] = up ? (x[b][e] - mx) + kKv4Top : x[b][e];
                }
                float pe[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    pe[e] = fast_exp2(x[b][e]);
                    s.l += pe[e];
                }
                if (big) kv4_pv<KV, D, true>(v[0], v[1], pe, s);
                else kv4_pv<KV, D, false>(v[0], v[1], pe, s);
            }
            kv4_load_v<D>(p, (const char *)p.v + (size_t)kvh_n * p.kv_head_stride, nx, lane, v);
            at = nx;
        }
        kv4_write<KV, D, R>(p, pc, lane, st);
        if (!has_next) break;
        pc = pn;
        ids = ids_n;
    }
}

// Two row blocks per wavefront for groups of 17 to 32 heads.
constexpr bool kv4_has_wide(int head_size) { return head_size <= 128; }

template <int KV, int D, int R>
static hipError_t launch_kv4_rows_of(const DecodeParams &p, hipStream_t st, hipEvent_t ev_start,
                                     hipEvent_t ev_stop) {
    const hipError_t e = launch_partition(
        paged_decode_partition_kv4_kernel<KV, D, R>, (unsigned)(p.num_waves / kKv4Waves), 64 * kKv4Waves,
        (size_t)(p.num_seqs + 1) * sizeof(int), st, ev_start, ev_stop, p, p.seq_lens, p.block_tables);
    if (e != hipSuccess) return e;
    return launch_merge<KV, D, kMfmaHeads * R, kKv4TileTokens>(p, st);
}

template <int KV, int D>
static hipError_t launch_kv4_size(const DecodeParams &p, int head_tile, hipStream_t st,
                                  hipEvent_t ev_start, hipEvent_t ev_stop) {
    if constexpr (kv4_has_wide(D))
        if (head_tile == 2 * kMfmaHeads) return launch_kv4_rows_of<KV, D, 2>(p, st, ev_start, ev_stop);
    return launch_kv4_rows_of<KV, D, 1>(p, st, ev_start, ev_stop);
}

template <int KV>
static hipError_t launch_kv4_dtype(const DecodeParams &p, int head_size, int head_tile, hipStream_t st,
                                   hipEvent_t ev_start, hipEvent_t ev_stop) {
    switch (head_size) {
#define XHIP_CASE(d) \
    case d: return launch_kv4_size<KV, d>(p, head_tile, st, ev_start, ev_stop);
        XHIP_FOR_HEAD_SIZES(XHIP_CASE)
#undef XHIP_CASE
    default: return hipErrorInvalidValue;
    }
}

template <int KV, int D> static const void *kv4_fn(int head_tile) {
    if constexpr (kv4_has_wide(D))
        if (head_tile == 2 * kMfmaHeads)
            return reinterpret_cast<const void *>(&paged_decode_partition_kv4_kernel<KV, D, 2>);
    return reinterpret_cast<const void *>(&paged_decode_partition_kv4_kernel<KV, D, 1>);
}

template <int KV> static int kv4_occupancy_dtype(int head_size, int head_tile, size_t lds_bytes) {
    const void *fn = nullptr;
    switch (head_size) {
#define XHIP_CASE(d) \
    case d: fn = kv4_fn<KV, d>(head_tile); break;
        XHIP_FOR_HEAD_SIZES(XHIP_CASE)
#undef XHIP_CASE
    default: return 0;
    }
    int blocks = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, fn, 64 * kKv4Waves, lds_bytes) != hipSuccess)
        return 0;
    return blocks;
}

}  // namespace xhip
