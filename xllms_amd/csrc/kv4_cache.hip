// Row kernels of a 4-bit K/V cache: rows quantised as they are written to
// their page slots, read back, and copied from slot to slot.
//
// A lane takes 8 channels of one row, of K and of V: piece c = 4g + q is
// channels 8c..8c+7, quarter q of group g, so the four lanes of an aligned
// quad hold a group and its range is two quad_perm steps.  A wavefront takes 16
// pieces (lane % 16) of four consecutive tokens (lane / 16).  A K piece is one
// word of the page.  A V piece is a byte of 4 words, since a V word holds 4
// tokens of 2 channels (kv4_layout.h): where the four tokens lie in one aligned
// quad of slots, as a prompt's do, each lane exchanges bytes with the other
// tokens' lanes and moves one whole word; else it moves 4 bytes.  (A lane per
// piece and 4 bytes each moved 32768 tokens of 8 kv heads of 128 channels, bf16,
// 176 MB, in 59 us to the cache and 41 us out of it; this takes 47 and 33.)
// Memory bounds it: 49152 tokens of 8 kv heads of 256 channels, fp16, out of
// the cache, 529 MB, take 127 us, 4.2 TB/s (a large copy reaches 5.1); the
// 16-bit rows go past the caches (137 us with ordinary stores).  Blocks of two
// wavefronts write 32768 tokens' rows 2 us sooner than blocks of four, and read
// as fast.
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

constexpr int kKv4RowBlock = 128;
constexpr long long kKv4MaxItems = (1LL << 29) - 1;  // four lanes each, a launch's lanes below 2^31

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
        __builtin_nontemporal_store((float_to_chunk<KV, 8>(x)), (u32x4 *)((char *)rows + i * 2));
    }
}

// x as the fp32 number that it is: a conversion to fp16 behind it is a rounding of
// its own (the compiler joins it with the product in one instruction, which
// rounds once).
__device__ __forceinline__ float rounded(float x) {
    asm("" : "+v"(x));
    return x;
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
    const _Float16 low = (_Float16)lo, step = (_Float16)rounded((hi - lo) * (1.0f / 15.0f));
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

// Bytes exchanged between the lanes of a piece's four tokens.  To the cache: a
// lane has byte e of pair e; lane k gets pair k's word, token t in byte
// kv4_v_byte(t).  From it: the reverse.
__device__ __forceinline__ uint32_t swap_bytes(uint32_t w, int lane, bool to_cache) {
    const int at = lane & 15, k = lane >> 4;
    const uint32_t a0 = __shfl(w, at), a1 = __shfl(w, at + 16), a2 = __shfl(w, at + 32),
                   a3 = __shfl(w, at + 48);
    const uint32_t b = (uint32_t)(to_cache ? k : kv4_v_byte(k));
    const uint32_t sel = b | (4 + b) << 8 | 0x0C0C0000u;  // byte b of either word
    return to_cache ? __builtin_amdgcn_perm(a2, a0, sel) | __builtin_amdgcn_perm(a3, a1, sel) << 16
                    : __builtin_amdgcn_perm(a1, a0, sel) | __builtin_amdgcn_perm(a3, a2, sel) << 16;
}

template <int KV, int OP>
__global__ __launch_bounds__(kKv4RowBlock) void kv4_rows_kernel(const Kv4RowParams p) {
    const int lane = threadIdx.x & 63, k = lane >> 4;
    const uint32_t i = (blockIdx.x * (kKv4RowBlock / 64) + (threadIdx.x >> 6)) * 16 + (lane & 15);
    const int ng = kv4_groups(p.head_size);
    const uint32_t item = i < p.items ? i : 0u;
    const uint32_t row = div_by(item, p.row_div);  // quad of tokens * kv heads + head
    const int c = (int)(item - row * (uint32_t)(4 * ng));
    const uint32_t quad = div_by(row, p.head_div);
    const int h = (int)(row - quad * (uint32_t)p.num_kv_heads);
    const int tok = p.tok0 + (int)quad * 4 + k;
    const bool in_range = i < p.items && tok < p.num_tokens;
    long long slot = -1;
    if (in_range) {
        if (p.slots) {
            slot = p.slots[tok];
        } else {
            const int pos = p.positions[tok];
            if (pos >= 0 && pos < p.max_ctx) {
                const int blk = p.block_tables[(size_t)tok * p.max_blocks + (pos >> p.bs_shift)];
                if (blk >= 0) slot = (long long)blk * p.block_size + (pos & (p.block_size - 1));
            }
        }
    }
    const bool live = slot >= 0;
    // the four tokens in one aligned quad of slots, in order
    const unsigned long long in_order = __ballot(live && (slot & 3) == k && slot - k == __shfl(slot, lane & 15));
    const bool whole = (in_order >> (lane & 15) & 0x0001000100010001ull) == 0x0001000100010001ull;
    const int g = c >> 2, q = c & 3;
    const bool piece_ok = live && 8 * c < p.head_size;
    int t;
    const size_t base = tile_at(p, ng, live ? slot : 0, h, &t);
    const int kw = kv4_k_word(ng, t, q, g);
    const int vw = kv4_v_word(ng, t >> 2, 4 * q + k, g);
    const int vb = kv4_v_word(ng, t >> 2, 4 * q, g) + kv4_v_byte(t & 3);
    const int vpair = 4 * ng;  // bytes from one channel pair's word to the next
    // the quad's lanes store one parameter of the group each: K step, K low, V step, V low
    const int param = q == 1 ? kv4_k_low(ng, t, g) : q == 3 ? kv4_v_low(ng, t, g) : kv4_step(ng, t, g);
    const size_t elem = ((size_t)tok * p.num_kv_heads + h) * p.head_size + (size_t)c * 8;
    char *kt = p.key_cache + base, *vt = p.value_cache + base;
    uint16_t *pt = (uint16_t *)((q < 2 ? kt : vt) + param);
    if constexpr (OP == KV4_WRITE) {
        // (lanes of skipped tokens go along, with nothing read or written: their
        // neighbours exchange with them)
        float x[8], y[8];
        if (piece_ok) {
            load_piece<KV>(p.key, elem, x);
            load_piece<KV>(p.value, elem, y);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = y[e] = 0.0f;
        }
        const Kv4Piece a = quantise(x, piece_ok);
        const Kv4Piece b = quantise(y, piece_ok);
        uint32_t w = 0, v = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            w |= a.code[2 * e] << (4 * e) | a.code[2 * e + 1] << (16 + 4 * e);
            v |= (b.code[2 * e] | b.code[2 * e + 1] << 4) << (8 * e);
        }
        const uint32_t mine = swap_bytes(v, lane, true);
        if (!live) return;
        *(uint32_t *)(kt + kw) = w;
        if (whole) {
            *(uint32_t *)(vt + vw) = mine;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) *(uint8_t *)(vt + vb + e * vpair) = (uint8_t)(v >> (8 * e));
        }
        *pt = q == 0 ? a.step : q == 1 ? a.low : q == 2 ? b.step : b.low;
    } else if constexpr (OP == KV4_READ) {
        uint32_t w = 0, v = 0, word = 0;
        float ks = 0.0f, kl = 0.0f, vs = 0.0f, vl = 0.0f;
        if (live) {
            w = *(const uint32_t *)(kt + kw);
            if (whole) {
                word = *(const uint32_t *)(vt + vw);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v |= (uint32_t)*(const uint8_t *)(vt + vb + e * vpair) << (8 * e);
            }
            // (one load each: a load per lane and four quad_perms were 8% slower
            // on rows of 256 channels)
            ks = half_bits(*(const uint16_t *)(kt + kv4_step(ng, t, g)));
            kl = half_bits(*(const uint16_t *)(kt + kv4_k_low(ng, t, g)));
            vs = half_bits(*(const uint16_t *)(vt + kv4_step(ng, t, g)));
            vl = half_bits(*(const uint16_t *)(vt + kv4_v_low(ng, t, g)));
        }
        const uint32_t mine = swap_bytes(word, lane, false);
        if (whole) v = mine;
        if (!piece_ok) return;
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[2 * e] = fmaf(ks, (float)(w >> (4 * e) & 15), kl);
            x[2 * e + 1] = fmaf(ks, (float)(w >> (16 + 4 * e) & 15), kl);
            y[2 * e] = fmaf(vs, (float)(v >> (8 * e) & 15), vl);
            y[2 * e + 1] = fmaf(vs, (float)(v >> (8 * e + 4) & 15), vl);
        }
        store_piece<KV>(p.key, elem, x);
        store_piece<KV>(p.value, elem, y);
    } else {
        const long long from = live ? p.src_slots[tok] : -1;
        if (from < 0) return;
        int u;
        const size_t src = tile_at(p, ng, from, h, &u);
        const char *ks = p.key_cache + src, *vs = p.value_cache + src;
        const int ub = kv4_v_word(ng, u >> 2, 4 * q, g) + kv4_v_byte(u & 3);
        *(uint32_t *)(kt + kw) = *(const uint32_t *)(ks + kv4_k_word(ng, u, q, g));
#pragma unroll
        for (int e = 0; e < 4; e++)
            *(uint8_t *)(vt + vb + e * vpair) = *(const uint8_t *)(vs + ub + e * vpair);
        const int from_param = q == 1 ? kv4_k_low(ng, u, g) : q == 3 ? kv4_v_low(ng, u, g) : kv4_step(ng, u, g);
        *pt = *(const uint16_t *)((q < 2 ? ks : vs) + from_param);
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
    const long long per_quad = (long long)p.num_kv_heads * pieces;  // items of 4 tokens
    if (p.num_tokens <= 0 || per_quad <= 0) return hipSuccess;
    if (per_quad > kKv4MaxItems) return hipErrorInvalidValue;
    p.row_div = div_magic((uint32_t)pieces);
    p.head_div = div_magic((uint32_t)p.num_kv_heads);
    const long long quads_per_launch = kKv4MaxItems / per_quad;
    const long long quads = ((long long)p.num_tokens + 3) / 4;
    constexpr int kPerBlock = kKv4RowBlock / 4;  // items
    for (long long q0 = 0; q0 < quads; q0 += quads_per_launch) {
        const long long n = quads - q0 < quads_per_launch ? quads - q0 : quads_per_launch;
        p.tok0 = (int)(4 * q0);
        p.items = (uint32_t)(n * per_quad);
        const unsigned grid = (unsigned)(((long long)p.items + kPerBlock - 1) / kPerBlock);
        const hipError_t e = op == KV4_WRITE  ? launch_rows<KV4_WRITE>(p, dtype, grid, stream)
                             : op == KV4_READ ? launch_rows<KV4_READ>(p, dtype, grid, stream)
                                              : launch_rows<KV4_COPY>(p, KV_F16, grid, stream);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace xhip
