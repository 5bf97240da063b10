// kv4.cu -- rotary positions and the paged 4-bit key/value cache: the table of
// angles, appending, reading back.  The layout and the number format are in
// kv4.cuh; attention over the cache is in attend.cu.
//
// klearu-llm's counterpart is its CPU attention half (crates/klearu-llm/src/
// model/kv_cache.rs holds f32 keys and values); the 4-bit pages are this
// engine's own.
#include "engine.h"
#include "kv4.cuh"

namespace kl {
namespace {

// table[p][i] = (cos, sin)(p * inv_freq[i]) * factor, angles and functions in
// 64 bits (a far position's angle has no fraction bits left in 32), held in 32.
__global__ void rope_table_kernel(const double* inv_freq, int pairs, int64_t n, float factor, float2* table) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n * pairs) return;
  double s, c;
  sincos((double)(i / pairs) * inv_freq[i % pairs], &s, &c);
  table[i] = make_float2((float)(c * factor), (float)(s * factor));
}

// Rotates lane-held dims [8 l, 8 l + 8) of the row at p: pairs (2i, 2i + 1)
// interleaved, else (i, i + rot / 2); dims from rot on stay.
__device__ __forceinline__ void rotate8(float* x, const __nv_bfloat16* p, bool vec, int l, int rot, bool interleaved,
                                        const float2* cs) {
  const int d0 = 8 * l;
  if (d0 >= rot) return;
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (d0 + 2 * i < rot) {  // rot is even
        const float2 a = cs[(d0 >> 1) + i];
        const float u = x[2 * i], v = x[2 * i + 1];
        x[2 * i] = fmaf(u, a.x, -__fmul_rn(v, a.y));
        x[2 * i + 1] = fmaf(v, a.x, __fmul_rn(u, a.y));
      }
    }
    return;
  }
  const int half = rot >> 1;
  if ((half & 7) == 0) {  // the eight partners are one aligned vector, and all on one side
    float y[8];
    const bool first = d0 < half;
    load8_bf16(p + (first ? d0 + half : d0 - half), vec, y);
    const float2* a = cs + (first ? d0 : d0 - half);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], a[i].x, __fmul_rn(first ? -y[i] : y[i], a[i].y));
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = d0 + i;
    if (d < rot) {
      const bool first = d < half;
      const float y = to_f(p[first ? d + half : d - half]);
      const float2 a = cs[first ? d : d - half];
      x[i] = fmaf(x[i], a.x, __fmul_rn(first ? -y : y, a.y));
    }
  }
}

struct AppendArgs {
  Kv4View cache;
  SeqView seq;
  const int32_t* positions;  // nullable
  const float2* table;       // nullable: no rotation
  int rot, interleaved;
  int64_t max_pos;
  int q_heads;  // 0: no queries
  HeadRows q, k, v, q_out;
  int* err;
};

constexpr int AP_NT = 256;

// One group of D / 8 lanes per head vector, 8 dims per lane; block = the head
// vectors [16 or 32 of them] of one token (q heads, then k, then v).  All
// traffic is the vectors themselves, so the kernel is bound by memory for
// prompts and by its chain of dependent loads (sequence, page, vector) for one
// token.
template <int D>
__global__ void __launch_bounds__(AP_NT) kv4_append_kernel(AppendArgs a) {
  constexpr int L = D / 8;           // lanes per vector
  constexpr int PER = AP_NT / L;     // vectors per block
  const int kh = a.cache.kv_heads, items = a.q_heads + 2 * kh;
  const int l = threadIdx.x % L, item = blockIdx.x * PER + threadIdx.x / L;
  const int t = blockIdx.y + blockIdx.z * 65535;
  if (t >= a.seq.num_tokens) return;
  const int b = find_seq(a.seq.cu_q, a.seq.num_seqs, t);
  if (b >= a.seq.num_seqs) return;  // behind the last sequence: left as it is
  bool bad = false;
  const int ps = a.cache.page_size;
  const SeqSpan s = seq_span(a.seq, b, ps, &bad);
  const int index = s.kv_len - s.q_len + (t - s.row);
  const int pos = a.positions ? a.positions[t] : index;
  int64_t page = -1;
  if (index >= 0) {
    page = a.seq.table[b * a.seq.table_ld + index / ps];
    if (page < 0 || page >= a.cache.num_pages) {
      bad = true;
      page = -1;
    }
  }
  bool live = index >= 0;  // a token in front of its sequence's first is padding: nothing stored, zero queries
  if (a.table && live && (pos < 0 || pos >= a.max_pos)) {
    bad = true;
    live = false;
  }
  if (bad && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(a.err, DERR_BOUNDS);
  if (item >= items) return;

  const bool is_q = item < a.q_heads, is_k = !is_q && item < a.q_heads + kh;
  const int head = is_q ? item : is_k ? item - a.q_heads : item - a.q_heads - kh;
  const HeadRows& in = is_q ? a.q : is_k ? a.k : a.v;
  const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(in.p) + t * in.token + head * in.head;
  const unsigned group = (L == 16 ? 0xffffu : 0xffu) << ((threadIdx.x & 31) / L * L);
  float x[8];
  if (is_q) {
    if (live) {
      load8_bf16(p + 8 * l, in.vec, x);
      if (a.table) rotate8(x, p, in.vec, l, a.rot, a.interleaved, a.table + (int64_t)pos * (a.rot >> 1));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
    __syncwarp(group);  // q_out may be q: every lane has read its partners
    store8_bf16(static_cast<__nv_bfloat16*>(a.q_out.p) + t * a.q_out.token + head * a.q_out.head + 8 * l, a.q_out.vec, x);
    return;
  }
  if (!live || page < 0) return;
  load8_bf16(p + 8 * l, in.vec, x);
  if (is_k && a.table) rotate8(x, p, in.vec, l, a.rot, a.interleaved, a.table + (int64_t)pos * (a.rot >> 1));
  float lo = x[0], hi = x[0];
  bool fin = finite_f(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    fin = fin && finite_f(x[i]);
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(group, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(group, hi, o));
  }
  fin = __all_sync(group, fin);
  // 8 bits for step and minimum: the codes are taken against the rounded values
  __nv_bfloat16 st = __float2bfloat16_rn(__fdiv_rn(hi - lo, 15.f)), mn = __float2bfloat16_rn(lo);
  float sf = to_f(st), mf = to_f(mn);
  if (!fin || !finite_f(sf) || !finite_f(mf)) {
    st = __ushort_as_bfloat16(0);
    mn = __ushort_as_bfloat16(0x7fff);
    sf = 0.f;
  }
  uint32_t w = 0;
  if (sf > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = fminf(fmaxf(rintf(__fdiv_rn(x[i] - mf, sf)), 0.f), 15.f);
      w |= (uint32_t)c << (4 * kv4_nibble(i));
    }
  }
  const int off = index % ps, tok = off & 15;
  unsigned char* tile = kv4_tile(a.cache, kv4_tile_bytes(D), page, head, off >> 4);
  const int code = is_k ? kv4_k_off<D>(tok, l) : kv4_codes(D) + kv4_v_off<D>(tok, l);
  *reinterpret_cast<uint32_t*>(tile + code) = w;
  if (l == 0) {
    const uint32_t pr = (uint32_t)__bfloat16_as_ushort(st) | ((uint32_t)__bfloat16_as_ushort(mn) << 16);
    *reinterpret_cast<uint32_t*>(tile + 2 * kv4_codes(D) + tok * 8 + (is_k ? 0 : 4)) = pr;
  }
}

struct ReadArgs {
  Kv4View cache;
  SeqView seq;
  HeadRows k, v;
  int* err;
};

// The values that the cached vectors of the call's tokens stand for; zeros
// where a token has no place in the cache.
template <int D>
__global__ void __launch_bounds__(AP_NT) kv4_read_kernel(ReadArgs a) {
  constexpr int L = D / 8, PER = AP_NT / L;
  const int kh = a.cache.kv_heads;
  const int l = threadIdx.x % L, item = blockIdx.x * PER + threadIdx.x / L;
  const int t = blockIdx.y + blockIdx.z * 65535;
  if (t >= a.seq.num_tokens) return;
  const int b = find_seq(a.seq.cu_q, a.seq.num_seqs, t);
  if (b >= a.seq.num_seqs) return;
  bool bad = false;
  const int ps = a.cache.page_size;
  const SeqSpan s = seq_span(a.seq, b, ps, &bad);
  const int index = s.kv_len - s.q_len + (t - s.row);
  int64_t page = -1;
  if (index >= 0) {
    page = a.seq.table[b * a.seq.table_ld + index / ps];
    if (page < 0 || page >= a.cache.num_pages) {
      bad = true;
      page = -1;
    }
  }
  if (bad && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(a.err, DERR_BOUNDS);
  if (item >= 2 * kh) return;
  const bool is_k = item < kh;
  const int head = is_k ? item : item - kh;
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (page >= 0) {
    const int off = index % ps, tok = off & 15;
    const unsigned char* tile = kv4_tile(a.cache, kv4_tile_bytes(D), page, head, off >> 4);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(
        tile + (is_k ? kv4_k_off<D>(tok, l) : kv4_codes(D) + kv4_v_off<D>(tok, l)));
    const uint32_t pr = *reinterpret_cast<const uint32_t*>(tile + 2 * kv4_codes(D) + tok * 8 + (is_k ? 0 : 4));
    const float sf = __uint_as_float(pr << 16), mf = __uint_as_float(pr & 0xffff0000u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((w >> (4 * kv4_nibble(i))) & 15u), sf, mf);
  }
  const HeadRows& o = is_k ? a.k : a.v;
  store8_bf16(static_cast<__nv_bfloat16*>(o.p) + t * o.token + head * o.head + 8 * l, o.vec, x);
}

dim3 token_grid(int items, int per, int tokens) {
  const int y = std::min(tokens, 65535);
  return dim3((unsigned)ceil_div(items, per), (unsigned)y, (unsigned)ceil_div(tokens, 65535));
}

}  // namespace

void launch_rope_table(const double* inv_freq, int pairs, int64_t n, float factor, float2* table, cudaStream_t st) {
  rope_table_kernel<<<(unsigned)ceil_div(n * pairs, 256), 256, 0, st>>>(inv_freq, pairs, n, factor, table);
  count_launch();
}

void launch_kv4_append(const Kv4View& cache, int D, const SeqView& seq, const int32_t* positions, const float2* table,
                       int rot, int interleaved, int64_t max_pos, int q_heads, const HeadRows& q, const HeadRows& k,
                       const HeadRows& v, const HeadRows& q_out, int* err, cudaStream_t st) {
  const AppendArgs a{cache, seq, positions, table, rot, interleaved, max_pos, q_heads, q, k, v, q_out, err};
  const dim3 grid = token_grid(q_heads + 2 * cache.kv_heads, AP_NT / (D / 8), seq.num_tokens);
  if (D == 128) kv4_append_kernel<128><<<grid, AP_NT, 0, st>>>(a);
  else kv4_append_kernel<64><<<grid, AP_NT, 0, st>>>(a);
  count_launch();
}

void launch_kv4_read(const Kv4View& cache, int D, const SeqView& seq, const HeadRows& k, const HeadRows& v, int* err,
                     cudaStream_t st) {
  const ReadArgs a{cache, seq, k, v, err};
  const dim3 grid = token_grid(2 * cache.kv_heads, AP_NT / (D / 8), seq.num_tokens);
  if (D == 128) kv4_read_kernel<128><<<grid, AP_NT, 0, st>>>(a);
  else kv4_read_kernel<64><<<grid, AP_NT, 0, st>>>(a);
  count_launch();
}

}  // namespace kl
