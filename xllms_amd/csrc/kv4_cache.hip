// Row kernels of a 4-bit K/V cache: rows quantised as they are written to
// their page slots, read back, and copied from slot to slot.
//
// A lane takes 8 channels of one row, of K and of V: piece c = 4g + q is
// channels 8c..8c+7, quarter q of group g, so the four lanes of an aligned
// quad hold a group and its range is two quad_perm steps.  A K piece is one
// word of the page; a V piece is 4 bytes of 4 words, since a V word holds 4
// tokens of 2 channels (kv4_layout.h).
// In fp32, and part of the format (a reader of the header can repeat it to the
// bit):
//   x' = x clamped to +-65504
//   low = fp16(min x'), step = fp16((max x' - min x') * fp32(1/15))
//   code = rint((x' - low) * (1 / step)) clamped to 0..15; 0 where step is 0
// A NaN in the group makes low and step NaN and the codes 0.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kv4_cache.h"
#include "kv4_layout.h"
#include "paged_decode_kernels.h"

namespace xhip {

constexpr int kKv4RowBlock = 64;  // one wavefront per workgroup
constexpr long long kKv4MaxLanes = (1LL << 31) - 1;

// 8 elements of a row piece, as fp32.
template <int KV> __device__ __forceinline__ void load_piece(const void *rows, size_t i, float (&x)[8]) {
    if constexpr (KV == KV_F32) {
        const f32x4 a = __builtin_nontemporal_load((const f32x4 *)((const float *)rows + i));
        const f32x4 b = __builtin_nontemporal_load((const f32x4 *)((const float *)rows + i) + 1);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = a[e], x[4 + e] = b[e];
    } else {
        chunk_to_float<KV, 8>(stream_load16((const char *)rows + i * 2), x);
    }
}

template <int KV> __device__ __forceinline__ void store_piece(void *rows, size_t i, const float (&x)[8]) {
    if constexpr (KV == KV_F32) {
        float *dst = (float *)rows + i;
        *(f32x4 *)dst = f32x4{x[0], x[1], x[2], x[3]};
        *(f32x4 *)(dst + 4) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        *(u32x4 *)((char *)rows + i * 2) = float_to_chunk<KV, 8>(x);
    }
}

// Codes, low and step of one group whose 8-channel pieces lie in the lanes of
// a quad (piece_ok: the piece is inside head_size; else its codes are 0).
struct Kv4Piece {
    uint32_t code[8];
    uint16_t low, step;  // fp16 bits
};

__device__ __forceinline__ Kv4Piece quantise(const float (&in)[8], bool piece_ok) {
    float x[8], lo = INFINITY, hi = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        nan |= in[e] != in[e];
        x[e] = fminf(fmaxf(in[e], -65504.0f), 65504.0f);
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
    }
    if (!piece_ok) {
        nan = false;
        lo = INFINITY;
        hi = -INFINITY;
    }
    lo = fminf(lo, dpp_mov<0xB1>(lo));
    hi = fmaxf(hi, dpp_mov<0xB1>(hi));
    lo = fminf(lo, dpp_mov<0x4E>(lo));
    hi = fmaxf(hi, dpp_mov<0x4E>(hi));
    const int lane = threadIdx.x & 63;
    nan = ((__ballot(nan) >> (lane & ~3)) & 15) != 0;
    const _Float16 low = (_Float16)lo, step = (_Float16)((hi - lo) * (1.0f / 15.0f));
    const float lowf = (float)low, stepf = (float)step;
    const float inv = 1.0f / stepf;
    const bool live = piece_ok && !nan && stepf > 0.0f;
    Kv4Piece r;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float c = fminf(fmaxf(rintf((x[e] - lowf) * inv), 0.0f), 15.0f);
        r.code[e] = live ? (uint32_t)c : 0u;
    }
    r.low = nan ? (uint16_t)0x7E00 : __builtin_bit_cast(uint16_t, low);
    r.step = nan ? (uint16_t)0x7E00 : __builtin_bit_cast(uint16_t, step);
    return r;
}

__device__ __forceinline__ float half_bits(uint16_t h) {
    return (float)__builtin_bit_cast(_Float16, h);
}

// Address of the tile that holds slot `slot` of kv head h, and the slot's
// token in it.
__device__ __forceinline__ size_t tile_at(const Kv4RowParams &p, int ng, long long slot, int h,
                                          int *token) {
    const long long blk = slot >> p.bs_shift;
    const int off = (int)(slot & (p.block_size - 1));
    *token = off & (kKv4Tile - 1);
    return (size_t)(blk * p.kv_block_stride + h * p.kv_head_stride) +
           (size_t)(off / kKv4Tile) * (size_t)(10 * kKv4Group * ng);
}

template <int KV, int OP>
__global__ __launch_bounds__(kKv4RowBlock) void kv4_rows_kernel(const Kv4RowParams p) {
    const uint32_t i = blockIdx.x * kKv4RowBlock + threadIdx.x;
    const bool in_range = i < p.lanes;
    const int ng = kv4_groups(p.head_size);
    const uint32_t row = div_by(in_range ? i : 0u, p.row_div);  // token * kv heads + head
    const int c = (int)((in_range ? i : 0u) - row * (uint32_t)(4 * ng));
    const uint32_t tok_l = div_by(row, p.head_div);
    const int h = (int)(row - tok_l * (uint32_t)p.num_kv_heads);
    const int tok = p.tok0 + (int)tok_l;
    long long slot;
    if (p.slots) {
        slot = p.slots[tok];
    } else {
        const int pos = p.positions[tok];
        slot = -1;
        if (pos >= 0 && pos < p.max_ctx) {
            const int blk = p.block_tables[(size_t)tok * p.max_blocks + (pos >> p.bs_shift)];
            if (blk >= 0) slot = (long long)blk * p.block_size + (pos & (p.block_size - 1));
        }
    }
    const int g = c >> 2, q = c & 3;
    const bool piece_ok = 8 * c < p.head_size;
    // (lanes of one quad share the row, so a skipped token's quad is skipped
    // whole, and the quads that go on are complete)
    if (!in_range || slot < 0) return;
    int t;
    const size_t base = tile_at(p, ng, slot, h, &t);
    const int kw = kv4_k_word(ng, t, q, g);
    const int vb = kv4_v_word(ng, t >> 2, 4 * q, g) + kv4_v_byte(t & 3);
    const int vpair = 4 * ng;  // bytes from one channel pair's word to the next
    const int at_step = kv4_step(ng, t, g), k_low = kv4_k_low(ng, t, g), v_low = kv4_v_low(ng, t, g);
    const size_t elem = ((size_t)tok * p.num_kv_heads + h) * p.head_size + (size_t)c * 8;
    char *kt = p.key_cache + base, *vt = p.value_cache + base;
    if constexpr (OP == KV4_WRITE) {
        float x[8], y[8];
        if (piece_ok) {
            load_piece<KV>(p.key, elem, x);
            load_piece<KV>(p.value, elem, y);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = y[e] = 0.0f;
        }
        const Kv4Piece a = quantise(x, piece_ok);
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) w |= a.code[2 * e] << (4 * e) | a.code[2 * e + 1] << (16 + 4 * e);
        *(uint32_t *)(kt + kw) = w;
        const Kv4Piece b = quantise(y, piece_ok);
#pragma unroll
        for (int e = 0; e < 4; e++)
            *(uint8_t *)(vt + vb + e * vpair) = (uint8_t)(b.code[2 * e] | b.code[2 * e + 1] << 4);
        if (q == 0) {
            *(uint16_t *)(kt + at_step) = a.step;
            *(uint16_t *)(kt + k_low) = a.low;
            *(uint16_t *)(vt + at_step) = b.step;
            *(uint16_t *)(vt + v_low) = b.low;
        }
    } else if constexpr (OP == KV4_READ) {
        if (!piece_ok) return;
        const uint32_t w = *(const uint32_t *)(kt + kw);
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = *(const uint8_t *)(vt + vb + e * vpair);
        const float ks = half_bits(*(const uint16_t *)(kt + at_step));
        const float kl = half_bits(*(const uint16_t *)(kt + k_low));
        const float vs = half_bits(*(const uint16_t *)(vt + at_step));
        const float vl = half_bits(*(const uint16_t *)(vt + v_low));
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[2 * e] = fmaf(ks, (float)(w >> (4 * e) & 15), kl);
            x[2 * e + 1] = fmaf(ks, (float)(w >> (16 + 4 * e) & 15), kl);
            y[2 * e] = fmaf(vs, (float)(v[e] & 15), vl);
            y[2 * e + 1] = fmaf(vs, (float)(v[e] >> 4), vl);
        }
        store_piece<KV>(p.key, elem, x);
        store_piece<KV>(p.value, elem, y);
    } else {
        const long long from = p.src_slots[tok];
        if (from < 0) return;
        int u;
        const size_t src = tile_at(p, ng, from, h, &u);
        const char *ks = p.key_cache + src, *vs = p.value_cache + src;
        const int ub = kv4_v_word(ng, u >> 2, 4 * q, g) + kv4_v_byte(u & 3);
        *(uint32_t *)(kt + kw) = *(const uint32_t *)(ks + kv4_k_word(ng, u, q, g));
#pragma unroll
        for (int e = 0; e < 4; e++)
            *(uint8_t *)(vt + vb + e * vpair) = *(const uint8_t *)(vs + ub + e * vpair);
        if (q == 0) {
            *(uint16_t *)(kt + at_step) = *(const uint16_t *)(ks + kv4_step(ng, u, g));
            *(uint16_t *)(kt + k_low) = *(const uint16_t *)(ks + kv4_k_low(ng, u, g));
            *(uint16_t *)(vt + at_step) = *(const uint16_t *)(vs + kv4_step(ng, u, g));
            *(uint16_t *)(vt + v_low) = *(const uint16_t *)(vs + kv4_v_low(ng, u, g));
        }
    }
}

template <int OP>
static hipError_t launch_rows(const Kv4RowParams &p, int dtype, unsigned grid, hipStream_t stream) {
    switch (dtype) {
    case KV_F16: kv4_rows_kernel<KV_F16, OP><<<grid, kKv4RowBlock, 0, stream>>>(p); break;
    case KV_BF16: kv4_rows_kernel<KV_BF16, OP><<<grid, kKv4RowBlock, 0, stream>>>(p); break;
    case KV_F32: kv4_rows_kernel<KV_F32, OP><<<grid, kKv4RowBlock, 0, stream>>>(p); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_kv4_rows(const Kv4RowParams &params, int op, int dtype, hipStream_t stream) {
    Kv4RowParams p = params;
    const int pieces = 4 * kv4_groups(p.head_size);
    const long long per_token = (long long)p.num_kv_heads * pieces;
    if (p.num_tokens <= 0 || per_token <= 0) return hipSuccess;
    if (per_token > kKv4MaxLanes) return hipErrorInvalidValue;
    p.row_div = div_magic((uint32_t)pieces);
    p.head_div = div_magic((uint32_t)p.num_kv_heads);
    const long long tok_per_launch = kKv4MaxLanes / per_token;
    for (long long t0 = 0; t0 < p.num_tokens; t0 += tok_per_launch) {
        const long long n = p.num_tokens - t0 < tok_per_launch ? p.num_tokens - t0 : tok_per_launch;
        p.tok0 = (int)t0;
        p.lanes = (uint32_t)(n * per_token);
        const unsigned grid = (unsigned)(((long long)p.lanes + kKv4RowBlock - 1) / kKv4RowBlock);
        const hipError_t e = op == KV4_WRITE  ? launch_rows<KV4_WRITE>(p, dtype, grid, stream)
                             : op == KV4_READ ? launch_rows<KV4_READ>(p, dtype, grid, stream)
                                              : launch_rows<KV4_COPY>(p, KV_F16, grid, stream);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace xhip
