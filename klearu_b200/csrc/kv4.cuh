// kv4.cuh -- the paged 4-bit key/value cache: layout and shared device code.
//
// A head vector x of D values (D = 64 or 128) is held as D codes of 4 bits, a
// step s and a minimum m (bf16 each): x ~ s * c + m with m = bf16(min x),
// s = bf16((max x - min x) / 15), c = clamp(rint((x - m) / s), 0, 15), c = 0
// where s is 0.  A vector with a value that is not finite is held as m = NaN.
// One step for each head vector (not for each channel) is what lets attention
// multiply the bare codes: s and m act on whole rows of the score and the
// probability matrix, after and before the tensor cores.
//
// The unit of the layout is a tile of 16 tokens of one head, contiguous:
//   [K codes 8 D bytes][V codes 8 D bytes][16 x (ks, km, vs, vm) bf16].
// A page is kv_heads x (page_size / 16) tiles.  Inside a tile the codes stand
// in the order in which the lanes of a warp want them as matrix fragments
// (lane = 4 g + t, g < 8, t < 4), each lane's share 16-byte aligned and a
// warp's 512 bytes contiguous, so reads neither waste sectors nor meet bank
// conflicts in shared memory:
//  K: lane (g, t) owns dims [t D/4, (t+1) D/4) of tokens g and g + 8;
//  V: lane (g, t) owns dims [g D/8, (g+1) D/8) of tokens 2t, 2t+1, 2t+8, 2t+9.
// A 32-bit word holds 8 consecutive dims: dim e stands in nibble e / 2 if even,
// 4 + e / 2 if odd, so that (word >> 4 i) & 0x000f000f is the pair (2i, 2i+1).
#pragma once

#include "common.cuh"

namespace kl {

constexpr int KV4_TILE = 16;  // tokens per tile
__host__ __device__ constexpr int kv4_codes(int D) { return 8 * D; }             // bytes of a tile's K (or V) codes
__host__ __device__ constexpr int kv4_tile_bytes(int D) { return 16 * D + 128; }  // multiple of 128

// Byte offset, inside the tile's K (V) codes, of the word with dims
// [8 l, 8 l + 8) of token tok (0 .. 15).
template <int D>
__device__ __forceinline__ int kv4_k_off(int tok, int l) {
  const int h = tok >> 3, g = tok & 7;
  if (D == 128) return h * 512 + g * 64 + l * 4;
  return g * 64 + (l >> 1) * 16 + h * 8 + (l & 1) * 4;
}
template <int D>
__device__ __forceinline__ int kv4_v_off(int tok, int l) {
  const int h = tok >> 3, t = (tok & 7) >> 1, o = tok & 1;
  if (D == 128) return h * 512 + (l >> 1) * 64 + t * 16 + o * 8 + (l & 1) * 4;
  return l * 64 + t * 16 + h * 8 + o * 4;
}
__device__ __forceinline__ int kv4_nibble(int e) { return (e >> 1) + ((e & 1) << 2); }  // e < 8

// The cache as kernels see it.
struct Kv4View {
  unsigned char* base;
  int64_t num_pages;
  int page_size, kv_heads;
  int tiles_per_page;  // page_size / 16
  // tile / tiles_per_page = umulhi(tile, magic) >> shift for tiles below 2^31: magic = ceil(2^(32 + shift) / d),
  // 2^shift < d <= 2^(shift + 1); d = 1: magic 0
  uint32_t magic, shift;
};
__host__ inline Kv4View kv4_view(unsigned char* base, int64_t num_pages, int page_size, int kv_heads) {
  Kv4View v{base, num_pages, page_size, kv_heads, page_size / KV4_TILE, 0, 0};
  const uint32_t d = (uint32_t)v.tiles_per_page;
  if (d > 1) {
    while ((2u << v.shift) < d) ++v.shift;
    v.magic = (uint32_t)((((uint64_t)1 << (32 + v.shift)) + d - 1) / d);
  }
  return v;
}
// The column of the page table that a sequence's tile of 16 tokens is in.
__device__ __forceinline__ int kv4_column(const Kv4View& c, int tile) {
  return c.magic ? (int)(__umulhi((uint32_t)tile, c.magic) >> c.shift) : tile;
}
__device__ __forceinline__ unsigned char* kv4_tile(const Kv4View& c, int tile_bytes, int64_t page, int head, int tile) {
  return c.base + ((page * c.kv_heads + head) * c.tiles_per_page + tile) * (int64_t)tile_bytes;
}

// Sequences of a call: sequence b's new tokens are rows cu_q[b] .. cu_q[b+1],
// the last of its kv_len[b] tokens; token i is in page page_table[b][i / page_size].
struct SeqView {
  const int32_t* cu_q;
  const int32_t* kv_len;
  const int32_t* table;
  int64_t table_ld;
  int width;  // pages per row of the table
  int num_seqs, num_tokens;
};

// Token rows of any two strides (elements), the last dimension contiguous.
struct HeadRows {
  void* p;
  int64_t token, head;
  int vec;  // every row starts on 16 bytes
};

// Attention over the cache (attend.cu): what a launch needs on the device, and
// what the host chooses its variant by.
struct AttendArgs {
  Kv4View cache;
  SeqView seq;
  int q_heads;
  HeadRows q, out;
  float scale;
  int window;       // 0: none
  float* scratch;   // attend_workspace() bytes, 16-byte aligned
  int* err;
};
struct AttendShape {
  int D, q_heads, kv_heads, num_seqs, num_tokens;
  int max_q, max_kv;  // of any sequence; hints: they choose the launch, not the result
  int window;
};

// #{ j in 1 .. n : cu[j] <= t } for non-decreasing cu: the sequence of token t.
// All 32 lanes take part; 32 probes a round.
__device__ __forceinline__ int find_seq(const int32_t* cu, int n, int t) {
  int lo = 0, hi = n;
  const int lane = threadIdx.x & 31;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int64_t j = lo + (int64_t)(lane + 1) * step;
    const int c = __popc(__ballot_sync(FULL, j <= hi && cu[j] <= t));
    lo += c * step;
    hi = min(hi, lo + step - 1);
  }
  return lo;
}

// A sequence's rows and tokens, held to what the call's arrays have room for;
// *bad where they had to be.  Row `row` is token `first`, whatever was cut off;
// tokens from kv_len on have no place.
struct SeqSpan {
  int row, q_len, first, kv_len;
};
__device__ __forceinline__ SeqSpan seq_span(const SeqView& s, int b, int page_size, bool* bad) {
  SeqSpan r;
  const int a = s.cu_q[b], e = s.cu_q[b + 1], n = s.kv_len[b];
  r.row = max(0, min(a, s.num_tokens));
  r.q_len = max(0, min(e, s.num_tokens) - r.row);
  r.first = (int)((uint32_t)max(0, n) - ((uint32_t)e - (uint32_t)r.row));  // a number where there are rows: 0 <= row < e
  r.kv_len = (int)max((int64_t)0, min((int64_t)n, (int64_t)s.width * page_size));
  *bad = r.row != a || r.q_len != e - a || r.kv_len != n;
  return r;
}

__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// 8 bf16 of a row; vec: 16-byte aligned
__device__ __forceinline__ uint4 load8_raw(const __nv_bfloat16* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
  return make_uint4((uint32_t)s[0] | (uint32_t)s[1] << 16, (uint32_t)s[2] | (uint32_t)s[3] << 16,
                    (uint32_t)s[4] | (uint32_t)s[5] << 16, (uint32_t)s[6] | (uint32_t)s[7] << 16);
}
// as f32
__device__ __forceinline__ void load8_bf16(const __nv_bfloat16* p, bool vec, float* x) {
  const uint4 r = load8_raw(p, vec);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void store8_raw(__nv_bfloat16* p, bool vec, uint4 v) {
  if (vec) {
    *reinterpret_cast<uint4*>(p) = v;
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  unsigned short* s = reinterpret_cast<unsigned short*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[2 * i] = (unsigned short)(w[i] & 0xffffu);
    s[2 * i + 1] = (unsigned short)(w[i] >> 16);
  }
}
__device__ __forceinline__ void store8_bf16(__nv_bfloat16* p, bool vec, const float* x) {
  store8_raw(p, vec, make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])));
}

}  // namespace kl
