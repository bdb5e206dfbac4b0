// Layout of the quantised K/V cache, shared by the kernels that write, read
// and attend over it.
//
// Codes stand in rows of head_dim * bits / 8 bytes, one row per (page, head,
// token of the page), so 16 consecutive tokens are one contiguous piece that a
// bulk copy brings to shared memory as it stands.  Inside a row the codes are
// ordered for the attention's matrix instructions (m16n8k16, thread (g, t) of
// a warp: g = lane / 4, t = lane % 4), and 16-byte pieces are exchanged by
// token so that a warp's reads meet no shared memory bank twice.
//
//   K is the left operand of the scores (rows = tokens, contraction over the
//   dimensions).  Step j of the contraction covers dimensions 16j .. 16j+15,
//   of which thread t holds 16j + 4t + {0,1,2,3}.  The row is four chunks, one
//   per t, each with t's dimensions of all steps in order; chunks longer than
//   16 bytes are cut into pieces of 16, pieces n of all chunks stand together
//   (64 bytes), and odd tokens exchange pieces 2n and 2n + 1.
//     4 bits: word w of a chunk holds steps 2w and 2w+1; dimension i of step
//             2w + o stands in nibble {0, 4, 2, 6}[i] + o.
//     8 bits: word j of a chunk holds step j; dimension i stands in byte
//             {0, 2, 1, 3}[i].
//   V is the left operand of the output (rows = dimensions, contraction over
//   the tokens), read by transposing 8 x 8 half words.  Row tile m covers
//   dimensions 16m .. 16m+15, of which thread g holds 16m + 2g + {0,1}.
//   A 16-byte piece is one half word per g:
//     4 bits: piece p holds tiles 2p and 2p+1: (tile 2p: dimensions 2g, 2g+1;
//             tile 2p+1: the same), four nibbles from the low bits up.
//     8 bits: piece p holds tile p, two bytes.
//   Piece p stands at place p ^ v_swizzle(token).
#pragma once

#include "floats.cuh"

namespace icx {

struct KvView {
  uint8_t* codes[2];    // K, V
  uint32_t* params[2];  // s (bf16) in the low half, lo (bf16) in the high half
  int64_t pages;
  int page_shift, heads, dim, bits, group, group_shift;
};

struct KvTokens {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;  // nullable: one token per sequence
  int64_t tokens;
  int batch, width;
};

// Checks both arguments and fills the device views; `what` names the operator
// in messages.
int kv_views(const char* what, const icx_kv_cache* cache, const icx_kv_tokens* where, KvView* view,
             KvTokens* tokens);

__device__ __forceinline__ float param_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float param_low(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// Sequence of packed row i: the b with cu[b] <= i < cu[b+1], or -1.  Whatever
// cu holds, b is within the batch.
__device__ __forceinline__ int kv_sequence(const KvTokens& w, int64_t i) {
  if (w.cu == nullptr) return i < w.batch ? (int)i : -1;
  int lo = 0, hi = w.batch;   // first b with cu[b+1] > i
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)w.cu[mid + 1] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo < w.batch && (int64_t)w.cu[lo] <= i ? lo : -1;
}

// Page of position p of sequence b, or -1 where the table gives none.
__device__ __forceinline__ int64_t kv_page(const KvView& c, const KvTokens& w, int b, int p) {
  const int n = p >> c.page_shift;
  if (n >= w.width) return -1;
  const int64_t page = w.table[(int64_t)b * w.width + n];
  return page >= 0 && page < c.pages ? page : -1;
}

// Row of (page, head, token of the page) in the codes and params buffers.
__device__ __forceinline__ int64_t kv_row(const KvView& c, int64_t page, int head, int p) {
  return (((page * c.heads) + head) << c.page_shift) + (p & ((1 << c.page_shift) - 1));
}

// Byte where word w of K chunk t stands in the row of a token.  ROW = bytes per
// row.
template <int ROW>
__device__ __forceinline__ int k_word_at(int token, int t, int w) {
  if (ROW == 32) return t * 8 + w * 4;
  const int piece = ROW == 64 ? 0 : (w >> 2) ^ (token & 1);
  return piece * 64 + t * 16 + (w & 3) * 4;
}
template <int ROW>
__device__ __forceinline__ int v_swizzle(int token) {
  return ROW == 32 ? (token >> 2) & 1 : ROW == 64 ? (token >> 1) & 3 : token & 7;
}

}  // namespace icx
