// Byte layout of a K/V cache held in 4 bits (the nxt_paged_kv4_* operators
// and nxt_paged_attention_kv4).
//
// A row (one token, one kv head) of head_size channels is cut into groups of
// 32; dp = head_size rounded up to whole groups, ng = dp / 32.  Each group has
// a 4-bit code per channel, and `low` and `step` in fp16:
//   value = low + step * code.
// A page of one kv head is block_size / 16 tiles of 16 tokens, 10 * dp bytes
// each (5/8 byte a channel), the same in the K and the V cache up to the order
// inside:
//   [0, 8 dp)      codes
//     K: [16 tokens][4 quarters][ng] words; the word of quarter q and group g
//        holds channels 32g + 8q + 0..7, channel 2i in nibble i and 2i + 1 in
//        nibble 4 + i.
//     V: [4 token quads][16 channel pairs][ng] words; the word of quad a, pair
//        r and group g holds channels 32g + 2r (low nibbles) and 32g + 2r + 1
//        (high nibbles) of tokens 4a..4a+3, token 4a + j in byte kv4_v_byte(j).
//   [8 dp, 9 dp)   steps, fp16 [4 token quads][ng][4 tokens]
//   [9 dp, 10 dp)  lows, fp16.  K: [16 tokens][ng] (ng 3: [16][2], then [16], so
//                  that no token's words straddle).  V: as the steps.
// That is the order in which the attention's matrix instructions take their
// operands: a lane's codes of a tile are ng consecutive words of K (its token,
// its 8 of each group's 32 channels) and of V (its 4 tokens, its 2 channels of
// each group), and two 4-bit codes 16 bits apart, masked out of a word, are a
// pair of fp16 numbers (subnormals: code * 2^-24, or code * 2^-20 from bits
// 4-7) without a conversion.  Every token owns whole bytes, so two tokens are
// never a race on one byte.
// Channels past head_size in the last group have code 0.
#pragma once

namespace xhip {

constexpr int kKv4Tile = 16;   // tokens of a tile
constexpr int kKv4Group = 32;  // channels of a group

constexpr int kv4_groups(int head_size) { return (head_size + kKv4Group - 1) / kKv4Group; }
constexpr int kv4_tile_bytes(int head_size) { return 10 * kKv4Group * kv4_groups(head_size); }

// Offsets inside a tile (token 0..15, quarter 0..3, pair 0..15, group < ng).
constexpr int kv4_k_word(int ng, int token, int quarter, int group) {
    return ((token * 4 + quarter) * ng + group) * 4;
}
constexpr int kv4_v_word(int ng, int quad, int pair, int group) {
    return ((quad * 16 + pair) * ng + group) * 4;
}
constexpr int kv4_v_byte(int j) { return ((j & 1) << 1) | (j >> 1); }  // 0, 2, 1, 3
constexpr int kv4_step(int ng, int token, int group) {
    return 256 * ng + (((token >> 2) * ng + group) * 4 + (token & 3)) * 2;
}
constexpr int kv4_k_low(int ng, int token, int group) {
    return 288 * ng + (ng != 3 ? (token * ng + group) * 2
                               : group < 2 ? (token * 2 + group) * 2 : 64 + token * 2);
}
constexpr int kv4_v_low(int ng, int token, int group) {
    return 288 * ng + (((token >> 2) * ng + group) * 4 + (token & 3)) * 2;
}

}  // namespace xhip
