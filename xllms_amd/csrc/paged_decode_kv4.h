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
//     each group.  The second sum is one more MFMA, A = lows (lane: group j), of
//     which row NG is ones: the sum of the weights as they went in.
//     Weights are scaled to at most 2^13, which keeps p * step clear of fp16's
//     subnormals: at 2^13 a step of up to 2 (values that span 30) leaves
//     p * step below 2^14.  Once a piece meets a larger step its weights are
//     scaled to at most 2^2 instead (steps end at 8734).
//     p and p * step go in as two fp16 parts, hi + lo (~22 bits), by packed
//     arithmetic: c = fp16(p_hi step), lo = fp16(p_lo step + (p_hi step - c)),
//     the difference exact in one fma; for a bf16 output, whose half step is
//     2^-8, as one (p and p * step rounded once each, 2^-11).
//
// Memory.  Each wavefront has two slots of LDS with a raw copy of a tile's four
// cache tiles (10 dp bytes each), which buffer loads to LDS fill two tiles
// ahead: the keys' half of a slot is refilled when the scores are done, the
// values' half after PV.  So each cache byte crosses the vector memory path
// once (a register load of the steps would read them 16 times), and a whole
// tile per wavefront stays in flight without registers.  The loads are inline
// assembly without register outputs, and the waits count them: the compiler's
// own waits for LDS loads in flight would drain them all.
//
// Per 32 tokens of a kv head at head_size 128 that is 5120 bytes, about 210
// vector instructions (fp16 in split columns) and 28 MFMAs (bf16 in whole
// columns: 19).  With everything in LDS already the two kinds take 72%
// and 28% of the time, one after the other: a wavefront's tile is a chain.  The
// fetches alone reach 5.9-6.1 TB/s, the kernel 5.4 over a large batch (256
// sequences of 512-8192 tokens, 32 / 8 heads of 128, fp16, 1.43 GB in 271 us with
// the merge); few tiles a wavefront leave the start (1.2 us of plan, 4 us to the
// first tile) and the end in sight (64 sequences of 512-4096: 43 us of kernel for
// 189 MB).  What did not help: three slots, three wavefronts a SIMD, one wavefront
// with 64-token tiles, wavefront priorities, ranges handed out by a counter, and
// the second fp16 parts of split columns in the spare columns (9 MFMAs fewer).
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
    static constexpr int kPieces = kBytes / 16;             // 16-byte pieces of a cache tile
    static constexpr int kFetches = (kPieces + 63) / 64;    // loads of a cache tile
    static constexpr int kLowWords = (NG + 1) / 2;          // a token's lows of K
    static constexpr int kOnes = 4 * kBytes;                // K a, K b, V a, V b, then eight ones
    static constexpr int kSlot = 4 * kBytes + 16;
    static constexpr int kHalfFetches = 2 * kFetches;       // loads of K (or V) of a tile
};

// Starts a cache tile's way to LDS address `lds`: nothing waits for it here.
// With ok false it touches no memory, and what LDS then holds is not used.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int D>
__device__ __forceinline__ void kv4_fetch(const char *tile, bool ok, uint32_t lds, int lane) {
    using G = Kv4Geometry<D>;
    const uint64_t at = (uint64_t)tile;
    // (uniform already; said once more where the assembly needs it)
    const u32x4 rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                        (uint32_t)__builtin_amdgcn_readfirstlane((int)((at >> 32) & 0xFFFFu)),
                        (uint32_t)__builtin_amdgcn_readfirstlane(ok ? G::kBytes : 0), 0x00020000u};
    lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
    const uint32_t off = (uint32_t)lane * 16;
#pragma unroll
    for (int c = 0; c < G::kFetches; c++) {
        constexpr int kLast = G::kPieces - 64 * (G::kFetches - 1);  // lanes of the last load
        if (c < G::kFetches - 1 || kLast == 64)
            asm volatile("s_mov_b32 m0, %0\n\t"
                         "s_nop 0\n\t"
                         "buffer_load_dwordx4 %1, %2, 0 offen offset:%3 nt lds"
                         :
                         : "s"(lds), "v"(off), "s"(rsrc), "n"(1024 * c)
                         : "memory", "m0");
        else  // (every lane is active here; a branch would end the scheduler's block)
            asm volatile("s_mov_b32 m0, %0\n\t"
                         "s_bfm_b64 exec, %4, 0\n\t"
                         "buffer_load_dwordx4 %1, %2, 0 offen offset:%3 nt lds\n\t"
                         "s_mov_b64 exec, -1"
                         :
                         : "s"(lds), "v"(off), "s"(rsrc), "n"(1024 * c), "n"(kLast)
                         : "memory", "m0");
    }
}
#pragma clang diagnostic pop

// Waits until at most N loads that were issued later are in flight.
template <int N> __device__ __forceinline__ void kv4_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

__device__ __forceinline__ f32x4 mfma_h(u32x4 a, u32x4 b, f32x4 c) {
    return mfma_qk<KV_F16>(a, b, c);
}

__device__ __forceinline__ uint32_t half_pair(float a, float b) { return pack16<KV_F16>(a, b); }

// What fp16 pair h leaves of two floats it was rounded from, as an fp16 pair
// (the differences are exact in fp32).
__device__ __forceinline__ uint32_t half_rest(float a, float b, uint32_t h) {
    uint32_t r;
    asm("v_fma_mixlo_f16 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(r) : "v"(a), "v"(h));
    asm("v_fma_mixhi_f16 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(r) : "v"(b), "v"(h));
    return r;
}

// x where ok, else -inf: in place, inside a rarely taken branch.
__device__ __forceinline__ void keep_score(float &x, bool ok) {
    const unsigned long long m = __ballot(ok);
    asm("v_cndmask_b32 %0, %1, %0, %2" : "+v"(x) : "v"(-INFINITY), "s"(m));
}

// Two codes of a word as fp16, times kv4_code_scale: nibbles 0 and 4, or with HIGH
// nibbles 1 and 5, which come 16 times as large.  The masked word is a pair of
// subnormals, code * 2^-24.  The matrix cores keep them, but align the products of
// an instruction by the exponents of their operands, of which a subnormal's is up
// to 10 above its leading bit: a sum is right to ~2^-19 of its largest product,
// always cut towards zero.  Under the rounding of a 16-bit output that goes;
// for fp32 they are made normal numbers first, which is one multiplication a word.
template <int KV> constexpr int kv4_code_exp() { return KV == KV_F32 ? 9 : 24; }
template <int KV> constexpr float kv4_code_scale() { return 1.0f / (1 << kv4_code_exp<KV>()); }

template <int KV, bool HIGH> __device__ __forceinline__ uint32_t code_pair(uint32_t w) {
    w &= HIGH ? 0x00f000f0u : 0x000f000fu;
    if constexpr (KV != KV_F32) return w;
    constexpr _Float16 k = 32768;
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w) * f16x2{k, k});
}

// Query operands of one head block.  kTerms: fp16 parts of a query element.
// SPLIT: head j & 7 in columns j and j + 8, and the operands of the two cache
// tiles: [0] is zero in columns 8-15, [1] in columns 0-7.
template <int KV, int D, bool SPLIT> struct Kv4Query {
    static constexpr int kTerms = KV == KV_F32 ? 2 : 1;
    static constexpr int kTiles = SPLIT ? 2 : 1;
    u32x4 q[kTiles][kTerms][Kv4Geometry<D>::NG];
    u32x2 sums[kTiles];  // the groups' sums, in fp16 parts hi (quarters 0, 1: groups 0-3,
                       // 4-7) and lo (quarters 2, 3)
    float a, b;        // score (log2 units) = a * (code part) + b * (low part)
};

template <int KV, int D, bool SPLIT>
__device__ __forceinline__ void kv4_load_query(const DecodeParams &p, const MfmaPiece &pc, int lane,
                                               int head0, int heads, Kv4Query<KV, D, SPLIT> &o) {
    using G = Kv4Geometry<D>;
    constexpr int NG = G::NG, EB = KvTraits<KV>::kBytes;
    const int j = lane & (SPLIT ? 7 : 15), q = lane >> 4;
    // in SPLIT, the operand of one cache tile
    const uint32_t first = !SPLIT || (lane & 8) == 0 ? ~0u : 0u;
    auto put = [&](u32x4 *to, u32x4 x) {  // to[tile * kTerms * NG]
        to[0] = x & first;
        if constexpr (SPLIT) to[Kv4Query<KV, D, SPLIT>::kTerms * NG] = x & ~first;
    };
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
    const bool row_bad = ((bad | bad >> 16 | bad >> 32 | bad >> 48) >> (lane & 15) & 1) != 0;
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
        put(&o.q[0][0][g], hi);
        if constexpr (KV == KV_F32) {
            u32x4 lo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const f32x2 r = unpack16<KV_F16>(lane_word(hi, e));
                lo[e] = half_pair(x[g][2 * e] - r.x, x[g][2 * e + 1] - r.y);
            }
            put(&o.q[0][1][g], lo);
        }
    }
    // A query with an infinity or NaN makes every score of its head NaN.
    if (row_bad) sum[0] = __builtin_nanf("");
    float s4[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float s0 = i < NG ? sum[i < NG ? i : 0] : 0.0f;
        const float s1 = 4 + i < NG ? sum[4 + i < NG ? 4 + i : 0] : 0.0f;
        s4[i] = q & 1 ? s1 : s0;
    }
    const uint32_t h01 = half_pair(s4[0], s4[1]), h23 = half_pair(s4[2], s4[3]);
    const f32x2 r01 = unpack16<KV_F16>(h01), r23 = unpack16<KV_F16>(h23);
    const u32x2 sums = q < 2 ? u32x2{h01, h23}
                             : u32x2{half_pair(s4[0] - r01.x, s4[1] - r01.y), half_pair(s4[2] - r23.x, s4[3] - r23.y)};
    o.sums[0] = sums & first;
    if constexpr (SPLIT) o.sums[1] = sums & ~first;
    o.a = __builtin_amdgcn_ldexpf(p.scale_log2, ex - 15 + kv4_code_exp<KV>());
    o.b = __builtin_amdgcn_ldexpf(p.scale_log2, ex - 15 + 9);
}

// The matrix cores cut what they add to an accumulator towards zero, and the two
// sums of PV have opposite signs: over many tiles in one range the sums drift.
// (32768 tokens of normal values under nearly equal weights, where the output is
// 1/360 of sum p (step code + |low|): fp16 outputs 4.3e-4 off, 1.9e-4 folded; fp32
// 5e-4 and 1.5e-4.)  fp32 outputs add each tile's products to the state by
// ordinary additions; fp16 ones move the sums to a second set of registers every
// kKv4FoldTiles tiles, where that set costs no wavefront per SIMD (not at head
// sizes 80 and 96: 24 sequences of 80, 30.5 us a step, 33.5 folded; 128: 54.4 and
// 54.9).  bf16 has a half step of 2^-8 and no need, two row blocks have no room.
constexpr int kKv4FoldTiles = 32;
template <int KV, int D, int R> constexpr bool kv4_fold() {
    return KV == KV_F16 && R == 1 && D != 80 && D != 96 && D != 192;
}
template <int KV, int R> constexpr bool kv4_add_tiles() { return KV == KV_F32 && R == 1; }

// Running state of one head block: lane (q, j) owns head j.
template <int D> struct Kv4State {
    f32x4 o[Kv4Geometry<D>::NG][2];  // [group][odd channel], rows 4q..4q+3: kv4_code_scale of it,
                                     // of the odd one 16 times that
    f32x4 low;                       // row 4q + i: group 4q + i's sum of p * low; row NG: the
                                     // sum of p
    float base;                      // weights of head j are 2^(score - base)
    float limit;                     // score - base from which the base moves; -inf (and
                                     // base 0) before the head's first score
};

// log2 of the largest weight a base lets through, before and after a piece
// meets a step of 2 or more (an fp16 of which a bit of kKv4BigStep is set).  A
// base that moves leaves the largest score kKv4Slack below it, so that the next
// few larger ones move nothing.
constexpr float kKv4Limit = 13.0f, kKv4BigLimit = 2.0f, kKv4Slack = 3.0f;
constexpr uint32_t kKv4BigStep = 0x40004000u;

template <int N> __device__ __forceinline__ void lds_words(const char *p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 x = *(const u32x4 *)(p + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; e++) w[i + e] = lane_word(x, e);
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const u32x2 x = *(const u32x2 *)(p + 4 * i);
            w[i] = x.x;
            w[i + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = *(const uint32_t *)(p + 4 * i);
    }
}

// What a lane's scores take of one cache tile's keys, out of LDS at t: the words
// of token j in quarter q, and its lows.
template <int D> struct Kv4Keys {
    uint32_t code[Kv4Geometry<D>::NG];
    u32x2 low;  // of this lane's quarter's groups
};

template <int D> __device__ __forceinline__ void kv4_keys(const char *t, int lane, Kv4Keys<D> &k) {
    using G = Kv4Geometry<D>;
    constexpr int NG = G::NG;
    const int j = lane & 15, q = lane >> 4;
    uint32_t low[G::kLowWords];
    lds_words(t + kv4_k_word(NG, j, q, 0), k.code);
    if constexpr (NG == 1) {
        low[0] = *(const uint16_t *)(t + kv4_k_low(NG, j, 0));
    } else if constexpr (NG == 3) {
        low[0] = *(const uint32_t *)(t + kv4_k_low(NG, j, 0));
        low[1] = *(const uint16_t *)(t + kv4_k_low(NG, j, 2));
    } else {
        lds_words(t + kv4_k_low(NG, j, 0), low);
    }
    k.low = u32x2{low[0], G::kLowWords > 1 ? low[G::kLowWords > 1 ? 1 : 0] : 0u};
    if constexpr (NG > 4) {
        k.low.x = q & 1 ? low[2] : k.low.x;
        k.low.y = q & 1 ? (G::kLowWords > 3 ? low[G::kLowWords > 3 ? 3 : 0] : 0u) : k.low.y;
    }
}

// The product of group g's codes of a cache tile with an operand set of a query
// block, added to c.
template <int KV, int D, bool SPLIT>
__device__ __forceinline__ f32x4 kv4_group(const Kv4Keys<D> &k, int g, const Kv4Query<KV, D, SPLIT> &qr,
                                           int tile, f32x4 c) {
    const uint32_t w = k.code[g], y = w >> 8;
    const u32x4 a = {code_pair<KV, false>(w), code_pair<KV, true>(w), code_pair<KV, false>(y), code_pair<KV, true>(y)};
    c = mfma_h(a, qr.q[tile][0][g], c);
    if constexpr (KV == KV_F32) c = mfma_h(a, qr.q[tile][1][g], c);
    return c;
}

// Scores of a tile's cache tiles (a at t, b behind it) against R head blocks,
// less each block's base (log2 units): x[b][0..3] of a's tokens 4q..4q+3 and
// x[b][4..7] of b's, head j.  SPLIT: x[b][0..3] of a in columns 0-7 and of b in
// columns 8-15.
template <int KV, int D, int R, bool SPLIT>
__device__ __forceinline__ void kv4_scores(const char *t, const Kv4Query<KV, D, SPLIT> (&qr)[R],
                                           const Kv4State<D> (&st)[R], int lane,
                                           float (&x)[R][SPLIT ? 4 : 8]) {
    using G = Kv4Geometry<D>;
    constexpr int NG = G::NG;
    const int q = lane >> 4;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    Kv4Keys<D> k[2];
    kv4_keys<D>(t, lane, k[0]);
    kv4_keys<D>(t + G::kBytes, lane, k[1]);
#pragma unroll
    for (int h = 0; h < (SPLIT ? 1 : 2); h++) {
        uint32_t step[2 * NG];
        lds_words(t + (SPLIT ? (lane & 8 ? G::kBytes : 0) : h * G::kBytes) + kv4_step(NG, 4 * q, 0), step);
#pragma unroll
        for (int b = 0; b < R; b++) {
            f32x4 lows = mfma_pv<KV_F16>(k[h].low, qr[b].sums[0], zero);
            if constexpr (SPLIT) lows = mfma_pv<KV_F16>(k[1].low, qr[b].sums[SPLIT ? 1 : 0], lows);
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < NG; g++) {
                f32x4 d = kv4_group<KV, D, SPLIT>(k[h], g, qr[b], 0, zero);
                if constexpr (SPLIT) d = kv4_group<KV, D, SPLIT>(k[1], g, qr[b], SPLIT ? 1 : 0, d);
                const f16x2 s01 = __builtin_bit_cast(f16x2, step[2 * g]);
                const f16x2 s23 = __builtin_bit_cast(f16x2, step[2 * g + 1]);
                s[0] = fmaf((float)s01.x, d[0], s[0]);
                s[1] = fmaf((float)s01.y, d[1], s[1]);
                s[2] = fmaf((float)s23.x, d[2], s[2]);
                s[3] = fmaf((float)s23.y, d[3], s[3]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                x[b][4 * h + i] = fmaf(qr[b].a, s[i], fmaf(qr[b].b, lows[i], -st[b].base));
        }
    }
}

// The values of one tile, out of LDS: of a, then of b.
template <int D> struct Kv4Values {
    uint32_t code[2][Kv4Geometry<D>::NG];      // tokens 4q..4q+3, channel pair j of each group
    uint32_t step[2][2 * Kv4Geometry<D>::NG];  // tokens 4q..4q+3 of each group
    uint32_t low[2][2];                        // tokens 4q..4q+3 of group j (row NG: ones)
};

// The word of the lane 8 columns on (j ^ 8).
__device__ __forceinline__ uint32_t other_half(uint32_t w) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x128, 0xF, 0xF, false);  // row_ror:8
}

// O += P V of one tile.  pe: the weights of the lane's tokens 4q..4q+3 of a,
// then of b.  SPLIT: of a in columns 0-7, which take b's from columns 8-15
// (whose own sums are of no use).
template <int KV, int D, int R, bool SPLIT>
__device__ __forceinline__ void kv4_pv(const Kv4Values<D> &v, const float (&pe)[R][SPLIT ? 4 : 8],
                                       Kv4State<D> (&st)[R]) {
    constexpr int NG = Kv4Geometry<D>::NG;
    constexpr bool kLo = KV != KV_BF16;  // a second fp16 part of the weights
    constexpr bool kAdd = kv4_add_tiles<KV, R>();
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 ph[R], pl[R];
    const u32x4 a = {v.low[0][0], v.low[0][1], v.low[1][0], v.low[1][1]};
#pragma unroll
    for (int b = 0; b < R; b++) {
#pragma unroll
        for (int i = 0; i < (SPLIT ? 2 : 4); i++) {
            const uint32_t h = half_pair(pe[b][2 * i], pe[b][2 * i + 1]);
            ph[b][i] = h;
            if constexpr (SPLIT) ph[b][i + 2] = other_half(h);
            if constexpr (kLo) {
                pl[b][i] = half_rest(pe[b][2 * i], pe[b][2 * i + 1], h);
                if constexpr (SPLIT) pl[b][i + 2] = other_half(pl[b][i]);
            }
        }
        f32x4 low = mfma_h(a, ph[b], kAdd ? zero : st[b].low);
        if constexpr (kLo) low = mfma_h(a, pl[b], low);
        st[b].low = kAdd ? st[b].low + low : low;
    }
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const uint32_t x = v.code[0][g], x8 = x >> 8, y = v.code[1][g], y8 = y >> 8;
        const u32x4 even = {code_pair<KV, false>(x), code_pair<KV, false>(x8), code_pair<KV, false>(y),
                            code_pair<KV, false>(y8)};
        const u32x4 odd = {code_pair<KV, true>(x), code_pair<KV, true>(x8), code_pair<KV, true>(y),
                           code_pair<KV, true>(y8)};
#pragma unroll
        for (int b = 0; b < R; b++) {
            u32x4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f16x2 s = __builtin_bit_cast(f16x2, v.step[i >> 1][2 * g + (i & 1)]);
                const f16x2 h = __builtin_bit_cast(f16x2, lane_word(ph[b], i));
                const f16x2 c = h * s;
                hi[i] = __builtin_bit_cast(uint32_t, c);
                if constexpr (kLo) {
                    const f16x2 l = __builtin_bit_cast(f16x2, lane_word(pl[b], i));
                    const f16x2 r = __builtin_elementwise_fma(h, s, -c);
                    lo[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(l, s, r));
                }
            }
            f32x4 o0 = mfma_h(even, hi, kAdd ? zero : st[b].o[g][0]);
            f32x4 o1 = mfma_h(odd, hi, kAdd ? zero : st[b].o[g][1]);
            if constexpr (kLo) {
                o0 = mfma_h(even, lo, o0);
                o1 = mfma_h(odd, lo, o1);
            }
            st[b].o[g][0] = kAdd ? st[b].o[g][0] + o0 : o0;
            st[b].o[g][1] = kAdd ? st[b].o[g][1] + o1 : o1;
        }
    }
}

// a += b, for every sum of a state.
template <int D> __device__ __forceinline__ void kv4_add_sums(Kv4State<D> &a, const Kv4State<D> &b) {
    a.low += b.low;
#pragma unroll
    for (int g = 0; g < Kv4Geometry<D>::NG; g++) {
        a.o[g][0] += b.o[g][0];
        a.o[g][1] += b.o[g][1];
    }
}
template <int D> __device__ __forceinline__ void kv4_scale_sums(Kv4State<D> &a, float f) {
    a.low *= f;
#pragma unroll
    for (int g = 0; g < Kv4Geometry<D>::NG; g++) {
        a.o[g][0] *= f;
        a.o[g][1] *= f;
    }
}
template <int D> __device__ __forceinline__ void kv4_zero_sums(Kv4State<D> &a) {
    a.low = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < Kv4Geometry<D>::NG; g++) a.o[g][0] = a.o[g][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// Row r of the state's low sums (the lane's head).
template <int D> __device__ __forceinline__ float kv4_low_row(const Kv4State<D> &st, int r, int lane) {
    const float own = st.low[r & 3];
    return __shfl(own, (r >> 2) * 16 + (lane & 15));
}

// The state's value of the lane's 8 channels of group g (32g + 8q..+7), not
// yet divided by l.
template <int KV, int D>
__device__ __forceinline__ void kv4_channels(const Kv4State<D> &st, int g, int lane, float (&f)[8]) {
    constexpr float kEven = 1.0f / kv4_code_scale<KV>();
    const float low = kv4_low_row<D>(st, g, lane);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f[2 * i] = fmaf(st.o[g][0][i], kEven, low);
        f[2 * i + 1] = fmaf(st.o[g][1][i], kEven / 16, low);
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
        const float l = kv4_low_row<D>(st[b], NG, lane);
        const int hj = 16 * b + j;
        const float mul = !pc.whole ? 1.0f : l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const size_t row = ((size_t)pc.slot * GT + hj) * D;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float f[8];
            kv4_channels<KV, D>(st[b], g, lane, f);
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

// Cut segments (wg_fix).  The wavefronts of a workgroup own consecutive ranges,
// so a segment's pieces in one workgroup are joined in it: a wavefront whose
// last piece continues its left neighbour's leaves its state in LDS, where the
// tiles were, and after a barrier the leftmost holder of each segment takes its
// neighbours' states, writes the rows if that was the whole segment, and else
// one partial.  (A cut first piece with others behind it, whose wavefront needs
// its slots still, goes to memory as a partial at once, and is taken from there.)
// (kv4_wg_fix: not with split columns, nor for two row blocks, whose states do
// not fit the slots.)
template <int D> struct Kv4FixSlot {
    f32x4 o[Kv4Geometry<D>::NG][2][64], low[64];
    float base[64], limit[64];
};

template <int D>
__device__ __forceinline__ void kv4_fix_store(Kv4FixSlot<D> &to, int lane, const Kv4State<D> &st) {
#pragma unroll
    for (int g = 0; g < Kv4Geometry<D>::NG; g++) {
        to.o[g][0][lane] = st.o[g][0];
        to.o[g][1][lane] = st.o[g][1];
    }
    to.low[lane] = st.low;
    to.base[lane] = st.base;
    to.limit[lane] = st.limit;
}

// Brings st to the larger of its base and another state's and returns the
// factor of that state's sums.  A state before its first score (limit -inf) has
// sums of zero, or of NaN, which stay.
template <int D> __device__ __forceinline__ float kv4_rebase(Kv4State<D> &st, float base, bool fresh) {
    const bool own_fresh = st.limit == -INFINITY;
    const float top = own_fresh ? base : fresh ? st.base : fmaxf(st.base, base);
    const float own = own_fresh ? 1.0f : fast_exp2(st.base - top);
    kv4_scale_sums<D>(st, own);
    st.base = top;
    if (!fresh) st.limit = 0.0f;  // (any but -inf: no more scores come)
    return fresh ? 1.0f : fast_exp2(base - top);
}

template <int D>
__device__ __forceinline__ void kv4_fix_absorb(const Kv4FixSlot<D> &from, int lane, Kv4State<D> &st) {
    const float w = kv4_rebase<D>(st, from.base[lane], from.limit[lane] == -INFINITY);
#pragma unroll
    for (int g = 0; g < Kv4Geometry<D>::NG; g++) {
        st.o[g][0] += from.o[g][0][lane] * w;
        st.o[g][1] += from.o[g][1][lane] * w;
    }
    st.low += from.low[lane] * w;
}

// The same from the partial in a slot of the workspace.
template <int KV, int D>
__device__ __forceinline__ void kv4_fix_absorb(const DecodeParams &p, const MfmaPiece &pc, int slot, int lane,
                                               Kv4State<D> &st) {
    constexpr int NG = Kv4Geometry<D>::NG;
    const int j = lane & 15, q = lane >> 4;
    if (j >= min(kMfmaHeads, p.group - pc.ht * kMfmaHeads)) return;  // (never written)
    const size_t row = (size_t)slot * kMfmaHeads + j;
    const float m = p.ws_ml[row * 2], l = p.ws_ml[row * 2 + 1];
    const float w = kv4_rebase<D>(st, m, m == -INFINITY);
    st.low[NG & 3] += q == NG >> 2 ? l * w : 0.0f;
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const int c = 32 * g + 8 * q;
        if (D % 32 != 0 && c >= D) continue;
        float f[8];
        load_floats(p.ws_o + row * D + c, f);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            st.o[g][0][i] += f[2 * i] * (w * kv4_code_scale<KV>());
            st.o[g][1][i] += f[2 * i + 1] * (w * (16 * kv4_code_scale<KV>()));
        }
    }
}

// One tile of a wavefront's range: where its two cache tiles are, in bytes from
// the start of either cache, and whether their pages are there.
struct Kv4TileRef {
    long long at_a, at_b;
    bool a, b;
};

// Walks the tiles of a wavefront's range, across its pieces, ahead of the
// computation.  Page ids are scalar loads, two tiles ahead: as vector loads they
// would be waited for behind every fetch in flight.
template <int D> struct Kv4Walker {
    RangeCursor cur;
    MfmaPiece pc;
    bool more;
    int t0;                  // first token of the next tile
    int blk[2], blk_then[2];  // page ids of its cache tiles, and of the tile behind it

    // Page id of the cache tile at token t of the piece (past its end: -1).
    __device__ __forceinline__ int id(const DecodeParams &p, const int *__restrict__ tables, int t) const {
        const int *bt = tables + (size_t)pc.s * p.max_blocks;
        const int b = bt[(t < pc.t_end ? t : pc.t_end - 1) >> p.bs_shift];
        return t < pc.t_end ? b : -1;
    }
    __device__ __forceinline__ void piece(const DecodeParams &p, const int *__restrict__ lens,
                                          const int *__restrict__ tables, const int *pre) {
        more = next_piece<kKv4TileTokens>(p, lens, pre, cur, pc);
        if (more) {
            t0 = pc.t_begin;
            for (int i = 0; i < 2; i++) {
                blk[i] = id(p, tables, t0 + kKv4Tile * i);
                blk_then[i] = id(p, tables, t0 + kKv4Tile * (2 + i));
            }
        }
    }
    __device__ __forceinline__ Kv4TileRef take(const DecodeParams &p, const int *__restrict__ lens,
                                               const int *__restrict__ tables, const int *pre) {
        if (!more) return Kv4TileRef{0, 0, false, false};
        const int blk_a = blk[0], blk_b = blk[1];
        constexpr unsigned kBytes = Kv4Geometry<D>::kBytes;
        const unsigned mask = (unsigned)p.block_size - 1;
        // (the strides are ints at the entry: 32-bit products)
        const long long head = (long long)pc.kvh * (int)p.kv_head_stride;
        const Kv4TileRef r = {
            head + (long long)blk_a * (int)p.kv_block_stride + ((((unsigned)t0 & mask) >> 4) * kBytes),
            head + (long long)blk_b * (int)p.kv_block_stride + ((((unsigned)t0 + 16 & mask) >> 4) * kBytes),
            blk_a >= 0, blk_b >= 0};
        t0 += kKv4TileTokens;
        if (t0 >= pc.t_end) {
            piece(p, lens, tables, pre);
        } else {
            for (int i = 0; i < 2; i++) {
                blk[i] = blk_then[i];
                blk_then[i] = id(p, tables, t0 + kKv4Tile * (2 + i));
            }
        }
        return r;
    }
};

// K (or V) of a tile into its half of an LDS slot.  Every LDS access so far has
// to be through: reads of the slot's last tile may be in the queue still, their
// uses scheduled past this point, and a page that is not there writes at once.
template <int D>
__device__ __forceinline__ void kv4_fetch_half(const void *cache, const Kv4TileRef &r, uint32_t lds, int lane) {
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    kv4_fetch<D>((const char *)cache + r.at_a, r.a, lds, lane);
    kv4_fetch<D>((const char *)cache + r.at_b, r.b, lds + Kv4Geometry<D>::kBytes, lane);
}

// Wavefronts per SIMD the kernel is compiled for, and LDS slots of each.
constexpr int kv4_waves_per_simd(int head_size) { return head_size > 192 ? 1 : 2; }
// (A third slot measured 1-2% slower, a third wavefront spilled.)
constexpr int kKv4Slots = 2;

// A wavefront computes one range of the plan.  (All of it stands in the kernel
// itself: the lengths and page ids are scalar loads only where the compiler sees
// that they come from the kernel's own restrict arguments.)
template <int KV, int D, int R, bool SPLIT>
__global__ __launch_bounds__(64 * kKv4Waves, (kv4_waves_per_simd(D))) void paged_decode_partition_kv4_kernel(
    const DecodeParams p, const int *__restrict__ lens, const int *__restrict__ tables) {
    using G = Kv4Geometry<D>;
    constexpr int TT = kKv4TileTokens, NG = G::NG, NF = G::kHalfFetches, S = kKv4Slots;
    constexpr int kX = SPLIT ? 4 : 8;  // scores of a lane
    static_assert(!SPLIT || R == 1, "split columns: one block");
    extern __shared__ int pre[];  // num_seqs + 1 split-unit prefixes
    constexpr bool kFold = kv4_fold<KV, D, R>();
    constexpr bool FIX = kv4_wg_fix(kMfmaHeads * R, SPLIT ? 1 : kMfmaHeads, D);
    // a wavefront's tiles, and its state at the end
    constexpr int kWaveLds = S * G::kSlot > (int)sizeof(Kv4FixSlot<D>) || !FIX ? S * G::kSlot : (int)sizeof(Kv4FixSlot<D>);
    __shared__ __attribute__((aligned(16))) char slots[kKv4Waves][kWaveLds];
    // what a wavefront has of its left neighbour's last segment: nothing, a state in
    // LDS that the next wavefront continues, one that ends the segment, or a partial
    // in memory (which ends it)
    enum { kNothing, kOpen, kEnd, kStored };
    __shared__ int continues[FIX ? kKv4Waves : 1];
    XHIP_WG_BEGIN(p);
    if (threadIdx.x < S * kKv4Waves)  // (the fetches leave them alone)
        *(u32x4 *)&slots[threadIdx.x / S][threadIdx.x % S * G::kSlot + G::kOnes] =
            u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
    batch_prefix<TT, kKv4Waves>(p, pre);
    XHIP_WG_STAMP(p, 1);
    const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int total = __builtin_amdgcn_readfirstlane(pre[p.num_seqs]);
    const int lb = logical_block(p, total);
    XHIP_WG_PUT(p, 3, lb);
    const int w = lb * kKv4Waves + wave;
    const int tpw = tiles_per_wave(total, p.num_waves, p.min_tiles_per_wave);
    if (blockIdx.x == 0 && threadIdx.x == 0) p.ws_prefix[p.num_seqs + 1] = tpw;  // for the merge
    const long long g_lo = (long long)w * tpw;
    RangeCursor cur;
    cur.g = (int)g_lo;
    cur.g_end = g_lo < total ? min(total, cur.g + tpw) : cur.g;
    cur.first = 1;
    cur.w = w;
    cur.ht = -1;
    cur.s = 0;
    if (g_lo < total) {
        int lo = 0, hi = p.num_seqs - 1;  // the sequence holding unit g
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= cur.g) lo = mid; else hi = mid - 1;
        }
        cur.s = __builtin_amdgcn_readfirstlane(lo);
    }
    const RangeCursor start = cur;
    MfmaPiece pc;
    bool has_next = next_piece<TT>(p, lens, pre, cur, pc);
    Kv4State<D> st[R];
    bool have_last = false;  // of a cut piece, in st
    int cont = kNothing;
    if (has_next) {
        Kv4Walker<D> ahead;
        ahead.cur = start;
        ahead.piece(p, lens, tables, pre);
        // LDS address of the wavefront's slots, K half then V half of each
        const uint32_t lds0 =
            (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)&slots[wave][0];
        Kv4TileRef ref[S];  // the tile at hand and those behind it
#pragma unroll
        for (int i = 0; i < S; i++) {
            ref[i] = ahead.take(p, lens, tables, pre);
            kv4_fetch_half<D>(p.k, ref[i], lds0 + i * G::kSlot, lane);
            kv4_fetch_half<D>(p.v, ref[i], lds0 + i * G::kSlot + 2 * G::kBytes, lane);
        }
        // the lane's lows of V: group j's, or past the groups the ones
        const int low_a = j < NG ? 2 * G::kBytes + kv4_v_low(NG, 4 * q, j < NG ? j : 0) : G::kOnes;
        const int low_b = j < NG ? low_a + G::kBytes : G::kOnes;
        int slot = 0;
        XHIP_WAVE_STAMP(p, wave, 0);
        while (has_next) {
            Kv4Query<KV, D, SPLIT> qr[R];
            const int g0 = pc.ht * kMfmaHeads * R;
            float limit = kKv4Limit;
            uint32_t big_step = kKv4BigStep;
#pragma unroll
            for (int b = 0; b < R; b++) {
                kv4_load_query<KV, D, SPLIT>(p, pc, lane, g0 + 16 * b, p.group - g0 - 16 * b, qr[b]);
                kv4_zero_sums<D>(st[b]);
                st[b].base = 0.0f;
                st[b].limit = -INFINITY;
            }
            Kv4State<D> past;  // (kFold: the sums of the tiles up to the last fold)
            if constexpr (kFold) kv4_zero_sums<D>(past);
            int fold_at = pc.t_begin + TT * kKv4FoldTiles;
            for (int t0 = pc.t_begin; t0 < pc.t_end; t0 += TT) {
                if (kFold && t0 == fold_at) {
                    fold_at += TT * kKv4FoldTiles;
                    kv4_add_sums<D>(past, st[0]);
                    kv4_zero_sums<D>(st[0]);
                }
                const Kv4TileRef nx = ahead.take(p, lens, tables, pre);
                char *ks = &slots[wave][slot * G::kSlot];
                const char *vs = ks + 2 * G::kBytes;
                const uint32_t lds = lds0 + (uint32_t)(slot * G::kSlot);
                float x[R][kX];
                kv4_wait<(2 * S - 1) * NF>();  // later: this tile's V, K and V of the next S - 1
                // tokens past the end or in missing pages (uniform, which the compiler
                // cannot see)
                const bool part = __builtin_amdgcn_readfirstlane(t0 + TT > pc.t_end || !ref[0].a || !ref[0].b);
                if (SPLIT && part) {
                    // a product of b's lows with the zeros of columns 0-7 is added to
                    // a's: no NaN there, whatever the slots hold
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int n = (h ? ref[0].b : ref[0].a) ? pc.t_end - t0 - 16 * h : 0;  // tokens
                        for (int i = lane; i < 16 * NG; i += 64)
                            if (i / NG >= n)
                                *(uint16_t *)(ks + h * G::kBytes + kv4_k_low(NG, i / NG, i % NG)) = 0;
                    }
                    wave_lds_fence();  // before the reads below, by other lanes
                }
                kv4_scores<KV, D, R, SPLIT>(ks, qr, st, lane, x);
                kv4_fetch_half<D>(p.k, nx, lds, lane);

                kv4_wait<(2 * S - 1) * NF>();  // later: K and V of the next S - 1, K of one more
                if (part) {
                    // no weight for such a token, and no step or low of its in a
                    // product.  In LDS, not in the registers: there the other way
                    // through the branch got a copy of every value.
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int n = (h ? ref[0].b : ref[0].a) ? pc.t_end - t0 - 16 * h : 0;  // tokens
                        if (!SPLIT || h == 0) {
                            // (SPLIT: the lane's scores are of the cache tile of its column)
                            const int n_b = ref[0].b ? pc.t_end - t0 - 16 : 0;
                            const int m = SPLIT && (lane & 8) ? n_b : n;
#pragma unroll
                            for (int e = 0; e < 4; e++)
#pragma unroll
                                for (int b = 0; b < R; b++) keep_score(x[b][4 * h + e], 4 * q + e < m);
                        }
                        uint16_t *t = (uint16_t *)(ks + (2 + h) * G::kBytes);
                        for (int i = lane; i < 16 * NG; i += 64) {
                            if ((i / (4 * NG)) * 4 + (i & 3) < n) continue;
                            t[kv4_step(NG, 0, 0) / 2 + i] = 0;
                            t[kv4_v_low(NG, 0, 0) / 2 + i] = 0;
                        }
                    }
                    wave_lds_fence();  // before the reads below, by other lanes
                }
                Kv4Values<D> v;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const char *t = vs + h * G::kBytes;
                    lds_words(t + kv4_v_word(NG, q, j, 0), v.code[h]);
                    lds_words(t + kv4_step(NG, 4 * q, 0), v.step[h]);
                    lds_words(ks + (h ? low_b : low_a), v.low[h]);
                }
                uint32_t steps = 0;
#pragma unroll
                for (int g = 0; g < 2 * NG; g++) steps |= v.step[0][g] | v.step[1][g];
                const bool big = __any((steps & big_step) != 0);
#pragma unroll
                for (int b = 0; b < R; b++) {
                    Kv4State<D> &s = st[b];
                    float mx = x[b][0];
#pragma unroll
                    for (int e = 1; e < kX; e++) mx = fmaxf(mx, x[b][e]);
                    if (big || __any(mx > s.limit)) {
                        if (big) limit = kKv4BigLimit;
                        if constexpr (SPLIT) mx = fmaxf(mx, __shfl_xor(mx, 8));
                        mx = fmaxf(mx, __shfl_xor(mx, 16));
                        mx = fmaxf(mx, __shfl_xor(mx, 32));
                        const bool fresh = s.limit == -INFINITY;
                        // the base moves where a score passes its limit, and where
                        // the limit falls
                        const bool move = mx > s.limit || (!fresh && s.limit != limit);
                        const float most = fresh ? mx : fmaxf(mx, s.limit);
                        const float top = limit - kKv4Slack;
                        const float down = move ? most - top : 0.0f;
                        const float alpha = fresh || !move ? 1.0f : fast_exp2(-down);
                        s.base += down;
                        s.limit = move ? limit : s.limit;
                        kv4_scale_sums<D>(s, alpha);
                        if constexpr (kFold) kv4_scale_sums<D>(past, alpha);
                        // (the largest weight is a power of two to the bit)
#pragma unroll
                        for (int e = 0; e < kX; e++) x[b][e] = move ? (x[b][e] - most) + top : x[b][e];
                    }
#pragma unroll
                    for (int e = 0; e < kX; e++) x[b][e] = fast_exp2(x[b][e]);
                }
                if (big) big_step = 0;
                kv4_pv<KV, D, R, SPLIT>(v, x, st);
                kv4_fetch_half<D>(p.v, nx, lds + 2 * G::kBytes, lane);
#pragma unroll
                for (int i = 0; i + 1 < S; i++) ref[i] = ref[i + 1];
                ref[S - 1] = nx;
                slot = slot + 1 == S ? 0 : slot + 1;
            }
            if constexpr (kFold) kv4_add_sums<D>(st[0], past);
            MfmaPiece next = pc;
            has_next = next_piece<TT>(p, lens, pre, cur, next);
            have_last = FIX && !has_next && !pc.whole;
            if (have_last) break;
            if (FIX && !pc.whole && pc.t_begin > 0) cont = kStored;
            kv4_write<KV, D, R>(p, pc, lane, st);
            pc = next;
        }
        XHIP_WAVE_STAMP(p, wave, 1);
        kv4_wait<0>();  // nothing of this wavefront's may reach LDS after its end
    }
    if constexpr (FIX) {
        if (have_last && wave > 0 && pc.t_begin > 0) {
            kv4_fix_store<D>(*(Kv4FixSlot<D> *)slots[wave], lane, st[0]);
            cont = pc.t_end < pc.L ? kOpen : kEnd;
            have_last = false;
        }
        if (lane == 0) continues[wave] = cont;
        __syncthreads();
        if (have_last) {
            bool ends = pc.t_end >= pc.L;
            for (int k = wave + 1; k < kKv4Waves && !ends; k++) {
                const int c = __builtin_amdgcn_readfirstlane(continues[k]);
                if (c == kStored)
                    kv4_fix_absorb<KV, D>(p, pc, (w - wave + k) * 2, lane, st[0]);
                else
                    kv4_fix_absorb<D>(*(const Kv4FixSlot<D> *)slots[k], lane, st[0]);
                ends = c != kOpen;
            }
            pc.whole = ends && pc.t_begin == 0;
            kv4_write<KV, D, R>(p, pc, lane, st);
        }
    }
    XHIP_WG_FLUSH(p);
}

// Two row blocks per wavefront for groups of 17 to 32 heads.
constexpr bool kv4_has_wide(int head_size) { return head_size <= 128; }

template <int KV, int D, int R, bool SPLIT>
static hipError_t launch_kv4_kernel(const DecodeParams &p, hipStream_t st, hipEvent_t ev_start,
                                    hipEvent_t ev_stop) {
    return launch_partition(paged_decode_partition_kv4_kernel<KV, D, R, SPLIT>,
                            (unsigned)(p.num_waves / kKv4Waves), 64 * kKv4Waves,
                            (size_t)(p.num_seqs + 1) * sizeof(int), st, ev_start, ev_stop, p, p.seq_lens,
                            p.block_tables);
}

// (split columns: the score products hold the heads twice, for a tile's two cache
// tiles, so that a lane has 4 scores and not 8)
template <int KV, int D>
static hipError_t launch_kv4_size(const DecodeParams &p, int head_tile, hipStream_t st,
                                  hipEvent_t ev_start, hipEvent_t ev_stop) {
    if constexpr (kv4_has_wide(D)) {
        if (head_tile == 2 * kMfmaHeads) {
            const hipError_t e = launch_kv4_kernel<KV, D, 2, false>(p, st, ev_start, ev_stop);
            if (e != hipSuccess) return e;
            return launch_merge<KV, D, 2 * kMfmaHeads, kKv4TileTokens>(p, st);
        }
    }
    hipError_t e;
    if constexpr (kv4_split(1, D))
        e = kv4_split(p.group, D) ? launch_kv4_kernel<KV, D, 1, true>(p, st, ev_start, ev_stop)
                                  : launch_kv4_kernel<KV, D, 1, false>(p, st, ev_start, ev_stop);
    else
        e = launch_kv4_kernel<KV, D, 1, false>(p, st, ev_start, ev_stop);
    if (e != hipSuccess) return e;
    return launch_merge<KV, D, kMfmaHeads, kKv4TileTokens>(p, st);
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

template <int KV, int D> static const void *kv4_fn(int head_tile, int group) {
    if constexpr (kv4_has_wide(D))
        if (head_tile == 2 * kMfmaHeads)
            return reinterpret_cast<const void *>(&paged_decode_partition_kv4_kernel<KV, D, 2, false>);
    if constexpr (kv4_split(1, D))
        if (kv4_split(group, D))
            return reinterpret_cast<const void *>(&paged_decode_partition_kv4_kernel<KV, D, 1, true>);
    return reinterpret_cast<const void *>(&paged_decode_partition_kv4_kernel<KV, D, 1, false>);
}

template <int KV> static int kv4_occupancy_dtype(int head_size, int head_tile, int group, size_t lds_bytes) {
    const void *fn = nullptr;
    switch (head_size) {
#define XHIP_CASE(d) \
    case d: fn = kv4_fn<KV, d>(head_tile, group); break;
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
