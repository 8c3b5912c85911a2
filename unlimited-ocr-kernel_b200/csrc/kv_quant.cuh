// kv_quant.cuh — layout of a KV cache held in 4 or 8 bits (host and device).
//
// A group is 32 consecutive dims of one head of one token's key (or value);
// it holds a code per dim, a step s and a least value m (both bf16), and
// stands for m + s * code.  A stored code is the code less the middle one (8 of
// 16, 128 of 256) in two's complement: its highest bit flipped.  The cache of one head of one sequence is a
// sequence of 32-token tiles, each one contiguous block
//
//   [key codes][key parameters][value codes][value parameters]
//
// so that a tile is one bulk copy.  Codes lie in the order in which a warp's
// 8-bit matrix fragments (m16n8k32) take them, one 16-byte load per lane and
// 512-byte plane, lane (g, j) = (lane / 4, lane % 4):
//   keys   (rows = tokens, k = dims):   word r of lane (g, j) is token g + 8 r,
//          dims 4j .. 4j+3 of the group's lower half (bytes); 4 bits: the same
//          byte's high nibble is the dim 16 above it; 8 bits: the upper half
//          has a plane of its own;
//   values (rows = dims, k = tokens):   bytes are tokens 4j .. 4j+3 of the
//          tile's lower or upper half; 4 bits: word 2 mb + half, low nibble
//          dim 16 mb + g, high nibble dim 16 mb + g + 8; 8 bits: a plane per
//          mb, word (upper 8 dims) + 2 half.
// So one token's codes never share a byte with another token's, and a push
// writes whole bytes.  A group's parameters are one word per token (s low, m
// high), at the lane that holds the token in the attention kernel.
#pragma once

#ifdef __CUDACC__
#define UOCR_HD __host__ __device__ __forceinline__
#else
#define UOCR_HD inline
#endif

namespace uocr {

constexpr int kKvqTile = 32;       // tokens per tile
constexpr int kKvqGroup = 32;      // dims per group
constexpr int kKvqMaxDim = 256;

struct KvqLayout {
  int heads, dim, groups, bits;
  int codes;         // bytes of a tile's key (or value) codes
  int half;          // bytes of a tile's keys (or values): codes + parameters
  int tile;          // bytes of a tile
  long long tiles;   // tiles per (sequence, head)
};

UOCR_HD KvqLayout kvq_layout(int heads, int dim, int bits, long long slots) {
  KvqLayout L;
  L.heads = heads;
  L.dim = dim;
  L.bits = bits;
  L.groups = (dim + kKvqGroup - 1) / kKvqGroup;
  L.codes = L.groups * 512 * (bits / 4);
  L.half = L.codes + L.groups * 128;
  L.tile = 2 * L.half;
  L.tiles = (slots + kKvqTile - 1) / kKvqTile;
  return L;
}

// What turns codes, byte by byte or nibble by nibble, into stored codes and back.
UOCR_HD constexpr unsigned kvq_flip(int bits) { return bits == 4 ? 0x88888888u : 0x80808080u; }

// Lane (and parameter word) of token t of a tile.
UOCR_HD int kvq_lane(int t) { return (t & 7) * 4 + (t >> 3); }

// Byte of the code of (token t of the tile, dim d) among the key codes; with
// 4 bits its nibble is 1 (high) for dims of the group's upper half.
UOCR_HD int kvq_key_byte(int t, int d, int bits) {
  const int grp = d >> 5, half = (d >> 4) & 1, j = (d >> 2) & 3;
  const int plane = bits == 4 ? grp : grp * 2 + half;
  return plane * 512 + ((t & 7) * 4 + j) * 16 + (t >> 3) * 4 + (d & 3);
}
UOCR_HD int kvq_key_nibble(int d) { return (d >> 4) & 1; }

// The same among the value codes; the high nibble is the upper 8 of 16 dims.
UOCR_HD int kvq_value_byte(int t, int d, int bits) {
  const int grp = d >> 5, mb = (d >> 4) & 1, g = d & 7, up = (d >> 3) & 1;
  const int half = t >> 4, j = (t >> 2) & 3;
  const int plane = bits == 4 ? grp : grp * 2 + mb;
  const int word = bits == 4 ? mb * 2 + half : up + 2 * half;
  return plane * 512 + (g * 4 + j) * 16 + word * 4 + (t & 3);
}
UOCR_HD int kvq_value_nibble(int d) { return (d >> 3) & 1; }

// Byte of the parameter word of (token t, group grp) behind the codes.
UOCR_HD int kvq_param_byte(int t, int grp) { return grp * 128 + kvq_lane(t) * 4; }

}  // namespace uocr
