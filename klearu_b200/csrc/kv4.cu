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

// How pairs lie: not at all; (2i, 2i + 1) with rot a multiple of 8; (i, i + rot
// / 2) with rot a multiple of 16; either kind of any even rot.
enum TurnMode { TURN_NONE, TURN_PAIRS, TURN_HALVES, TURN_ANY };

// cos and sin of the pairs that dims [8 l, 8 l + 8) belong to, loaded ahead of
// their use: four pairs interleaved, else eight.
struct Turn {
  float2 cs[8];
};
template <int MODE>
__device__ __forceinline__ void load_turn(Turn& t, const float2* row, int l, int rot, bool interleaved) {
  const int d0 = 8 * l, half = rot >> 1;
  if (MODE == TURN_PAIRS || MODE == TURN_HALVES) {
    if (d0 >= rot) return;
    const float4* p = reinterpret_cast<const float4*>(row + (MODE == TURN_PAIRS ? 4 * l : d0 < half ? d0 : d0 - half));
#pragma unroll
    for (int i = 0; i < (MODE == TURN_PAIRS ? 2 : 4); ++i) *reinterpret_cast<float4*>(&t.cs[2 * i]) = p[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = interleaved ? d0 + 2 * i : d0 + i;
    t.cs[i] = make_float2(1.f, 0.f);
    if ((!interleaved || i < 4) && d < rot) t.cs[i] = row[interleaved ? d >> 1 : d < half ? d : d - half];
  }
}
// Turns lane-held dims [8 l, 8 l + 8) of the row at p; dims from rot on stay.
// All lanes of the row's group take part.
template <int MODE>
__device__ __forceinline__ void turn8(float* x, const Turn& t, const __nv_bfloat16* p, int l, int rot, bool interleaved,
                                      unsigned group) {
  const int d0 = 8 * l, half = rot >> 1;
  if (MODE == TURN_PAIRS || (MODE == TURN_ANY && interleaved)) {
    if (MODE == TURN_PAIRS && d0 >= rot) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = t.cs[i];
      const float u = x[2 * i], v = x[2 * i + 1];
      x[2 * i] = fmaf(u, a.x, -__fmul_rn(v, a.y));
      x[2 * i + 1] = fmaf(v, a.x, __fmul_rn(u, a.y));
    }
  } else if (MODE == TURN_HALVES) {  // the eight partners are another lane's, all on one side
    const bool first = d0 < half;
    const int from = d0 >= rot ? l : first ? l + (half >> 3) : l - (half >> 3);
    const int lane = ((threadIdx.x & 31) & ~(__popc(group) - 1)) + from;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = __shfl_sync(group, x[i], lane);
      if (d0 < rot) x[i] = fmaf(x[i], t.cs[i].x, __fmul_rn(first ? -y : y, t.cs[i].y));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + i;
      if (d < rot) {
        const bool first = d < half;
        const float y = to_f(p[first ? d + half : d - half]);
        x[i] = fmaf(x[i], t.cs[i].x, __fmul_rn(first ? -y : y, t.cs[i].y));
      }
    }
  }
}

constexpr int AP_NT = 256;
constexpr int AP_TOKENS = 4;  // tokens of a block, each looked up by a warp

// Where a token stands: its page and place in it, its position.
struct Place {
  int64_t page;  // -1: nowhere
  int off, pos;
  int kind;  // 0: of no sequence, left as it is; 1: padding or bad, zeros; 2: live
};
// By a warp.  *bad: something had to be left out.
__device__ __forceinline__ Place find_place(const Kv4View& cache, const SeqView& seq, const int32_t* positions, int t,
                                            bool table, int64_t max_pos, bool* bad) {
  Place r{-1, 0, 0, 0};
  const int b = find_seq(seq.cu_q, seq.num_seqs, t);
  if (b >= seq.num_seqs) return r;
  const SeqSpan s = seq_span(seq, b, cache.page_size, bad);
  const int index = s.kv_len - s.q_len + (t - s.row);
  r.pos = positions ? positions[t] : index;
  r.kind = 1;
  if (index < 0) return r;  // in front of its sequence's first token: padding
  const int col = kv4_column(cache, index >> 4);
  r.off = index - col * cache.page_size;
  r.page = seq.table[b * seq.table_ld + col];
  if (r.page < 0 || r.page >= cache.num_pages) {
    *bad = true;
    r.page = -1;
  }
  r.kind = 2;
  if (table && (r.pos < 0 || r.pos >= max_pos)) {
    *bad = true;
    r.kind = 1;
  }
  return r;
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
  int tokens;  // of a block
  int* err;
};

// The codes of the definition, quotients rounded as f32 divisions.
__device__ __noinline__ uint32_t exact_codes(float4 a, float4 b, float m, float s) {
  const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(x[i] - m, s)), 0.f), 15.f) << (4 * kv4_nibble(i));
  return w;
}
// By a reciprocal: quotients off by at most 2^-23 of 15 decide unless one is
// within 1e-5 of a border between two codes (or the reciprocal is none to use).
__device__ __forceinline__ uint32_t codes8(const float* x, float m, float s) {
  const float inv = __frcp_rn(s);
  uint32_t w = 0;
  bool near = !(s > 1e-30f && s < 1e30f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = fminf(fmaxf((x[i] - m) * inv, 0.f), 15.f), c = y + 8388608.f;  // 2^23: rounds to a whole number
    near = near || fabsf(y - (c - 8388608.f)) > 0.49999f;
    w |= (__float_as_uint(c) & 15u) << (4 * kv4_nibble(i));
  }
  return near ? exact_codes(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), m, s) : w;
}

// One group of D / 8 lanes per head vector, 8 dims per lane: a block's groups
// take 16 (D = 128) or 32 head vectors, q heads then k then v, of up to four
// tokens, two tokens' loads in flight at once.  All traffic is the vectors
// themselves: memory bounds it for prompts, the chain of dependent loads
// (sequence, page and position, vector) for one token.
template <int D, int MODE>
__global__ void __launch_bounds__(AP_NT, 3) kv4_append_kernel(AppendArgs a) {
  constexpr int L = D / 8;        // lanes per vector
  constexpr int PER = AP_NT / L;  // vectors per block
  constexpr int U = 2;            // tokens in flight
  __shared__ Place places[AP_TOKENS];
  const int kh = a.cache.kv_heads, items = a.q_heads + 2 * kh;
  const int l = threadIdx.x % L, item = blockIdx.x * PER + threadIdx.x / L;
  const int t0 = (int)(((int64_t)blockIdx.z * 65535 + blockIdx.y) * a.tokens);
  const int n = min(a.tokens, a.seq.num_tokens - t0);
  if ((int)(threadIdx.x >> 5) < n) {
    bool bad = false;
    const Place p = find_place(a.cache, a.seq, a.positions, t0 + (threadIdx.x >> 5), MODE != TURN_NONE, a.max_pos, &bad);
    if ((threadIdx.x & 31) == 0) places[threadIdx.x >> 5] = p;
    if (bad && (threadIdx.x & 31) == 0 && blockIdx.x == 0) atomicOr(a.err, DERR_BOUNDS);
  }
  const bool is_q = item < a.q_heads, is_k = !is_q && item < a.q_heads + kh;
  const int head = is_q ? item : is_k ? item - a.q_heads : item - a.q_heads - kh;
  const HeadRows& in = is_q ? a.q : is_k ? a.k : a.v;
  const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(in.p) + (int64_t)t0 * in.token + head * in.head;
  const int64_t stride = in.token;
  const bool vec = in.vec;
  const unsigned group = (L == 16 ? 0xffffu : 0xffu) << ((threadIdx.x & 31) / L * L);
  const bool turned = MODE != TURN_NONE && (is_q || is_k);
  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)  // the first ones before their places are known
    if (item < items && u < n) raw[u] = load8_raw(row + u * stride + 8 * l, vec);
  __syncthreads();
  if (item >= items) return;

  for (int u0 = 0; u0 < n; u0 += U) {
    Turn turn[U];
    if (u0 > 0) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u0 + u < n) raw[u] = load8_raw(row + (u0 + u) * stride + 8 * l, vec);
    }
    if (turned) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u0 + u < n && places[u0 + u].kind == 2)
          load_turn<MODE>(turn[u], a.table + (int64_t)places[u0 + u].pos * (a.rot >> 1), l, a.rot, a.interleaved);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u0 + u >= n) break;
      const Place& pl = places[u0 + u];
      const int kind = pl.kind;
      if (kind == 0 || (!is_q && (kind != 2 || pl.page < 0))) continue;
      float x[8];
      const uint32_t w4[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w4[i] << 16);
        x[2 * i + 1] = __uint_as_float(w4[i] & 0xffff0000u);
      }
      if (turned && kind == 2) turn8<MODE>(x, turn[u], row + (u0 + u) * stride, l, a.rot, a.interleaved, group);
      if (is_q) {
        if (kind != 2) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = 0.f;
        }
        __syncwarp(group);  // q_out may be q: every lane has read its partners
        store8_bf16(static_cast<__nv_bfloat16*>(a.q_out.p) + (int64_t)(t0 + u0 + u) * a.q_out.token + head * a.q_out.head +
                        8 * l,
                    a.q_out.vec, x);
        continue;
      }
      float lo = fminf(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), fminf(fminf(x[4], x[5]), fminf(x[6], x[7])));
      float hi = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      // 0 * x is 0 for a finite x, else NaN
      const float z = 0.f * x[0] + 0.f * x[1] + 0.f * x[2] + 0.f * x[3] + 0.f * x[4] + 0.f * x[5] + 0.f * x[6] + 0.f * x[7];
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(group, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(group, hi, o));
      }
      const bool fin = __all_sync(group, z == 0.f);
      // 8 bits for step and minimum: the codes are taken against the rounded values
      __nv_bfloat16 st = __float2bfloat16_rn(__fdiv_rn(hi - lo, 15.f)), mn = __float2bfloat16_rn(lo);
      float sf = to_f(st), mf = to_f(mn);
      if (!fin || !finite_f(sf) || !finite_f(mf)) {
        st = __ushort_as_bfloat16(0);
        mn = __ushort_as_bfloat16(0x7fff);
        sf = 0.f;
      }
      const uint32_t w = sf > 0.f ? codes8(x, mf, sf) : 0u;
      const int tok = pl.off & 15;
      unsigned char* tile = kv4_tile(a.cache, kv4_tile_bytes(D), pl.page, head, pl.off >> 4);
      const int code = is_k ? kv4_k_off<D>(tok, l) : kv4_codes(D) + kv4_v_off<D>(tok, l);
      *reinterpret_cast<uint32_t*>(tile + code) = w;
      if (l == 0) {
        const uint32_t pr = (uint32_t)__bfloat16_as_ushort(st) | ((uint32_t)__bfloat16_as_ushort(mn) << 16);
        *reinterpret_cast<uint32_t*>(tile + 2 * kv4_codes(D) + tok * 8 + (is_k ? 0 : 4)) = pr;
      }
    }
  }
}

struct ReadArgs {
  Kv4View cache;
  SeqView seq;
  HeadRows k, v;
  int tokens;  // of a block
  int* err;
};

// The values that the cached vectors of the call's tokens stand for; zeros
// where a token has no place in the cache.
template <int D>
__global__ void __launch_bounds__(AP_NT) kv4_read_kernel(ReadArgs a) {
  constexpr int L = D / 8, PER = AP_NT / L, U = 4;
  __shared__ Place places[AP_TOKENS];
  const int kh = a.cache.kv_heads;
  const int l = threadIdx.x % L, item = blockIdx.x * PER + threadIdx.x / L;
  const int t0 = (int)(((int64_t)blockIdx.z * 65535 + blockIdx.y) * a.tokens);
  const int n = min(a.tokens, a.seq.num_tokens - t0);
  if ((int)(threadIdx.x >> 5) < n) {
    bool bad = false;
    const Place p = find_place(a.cache, a.seq, nullptr, t0 + (threadIdx.x >> 5), false, 0, &bad);
    if ((threadIdx.x & 31) == 0) places[threadIdx.x >> 5] = p;
    if (bad && (threadIdx.x & 31) == 0 && blockIdx.x == 0) atomicOr(a.err, DERR_BOUNDS);
  }
  __syncthreads();
  if (item >= 2 * kh) return;
  const bool is_k = item < kh;
  const int head = is_k ? item : item - kh;
  const HeadRows o = is_k ? a.k : a.v;
  for (int u0 = 0; u0 < n; u0 += U) {
    uint32_t w[U], pr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = pr[u] = 0;
      if (u0 + u >= n || places[u0 + u].page < 0) continue;
      const Place pl = places[u0 + u];
      const int tok = pl.off & 15;
      const unsigned char* tile = kv4_tile(a.cache, kv4_tile_bytes(D), pl.page, head, pl.off >> 4);
      w[u] = *reinterpret_cast<const uint32_t*>(tile + (is_k ? kv4_k_off<D>(tok, l) : kv4_codes(D) + kv4_v_off<D>(tok, l)));
      pr[u] = *reinterpret_cast<const uint32_t*>(tile + 2 * kv4_codes(D) + tok * 8 + (is_k ? 0 : 4));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u0 + u >= n || places[u0 + u].kind == 0) continue;
      const float sf = __uint_as_float(pr[u] << 16), mf = __uint_as_float(pr[u] & 0xffff0000u);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((w[u] >> (4 * kv4_nibble(i))) & 15u), sf, mf);
      store8_bf16(static_cast<__nv_bfloat16*>(o.p) + (int64_t)(t0 + u0 + u) * o.token + head * o.head + 8 * l, o.vec, x);
    }
  }
}

// Four tokens a block where there are blocks enough, one where latency counts.
int block_tokens(int items, int per, int tokens) { return ceil_div(items, per) * tokens >= 4 * 1184 ? AP_TOKENS : 1; }
dim3 token_grid(int items, int per, int tokens, int each) {
  const int64_t n = ceil_div(tokens, each);
  return dim3((unsigned)ceil_div(items, per), (unsigned)std::min<int64_t>(n, 65535), (unsigned)ceil_div(n, 65535));
}

template <int D>
void launch_append(const AppendArgs& a, dim3 grid, cudaStream_t st) {
  if (!a.table) kv4_append_kernel<D, TURN_NONE><<<grid, AP_NT, 0, st>>>(a);
  else if (a.interleaved && a.rot % 8 == 0) kv4_append_kernel<D, TURN_PAIRS><<<grid, AP_NT, 0, st>>>(a);
  else if (!a.interleaved && a.rot % 16 == 0) kv4_append_kernel<D, TURN_HALVES><<<grid, AP_NT, 0, st>>>(a);
  else kv4_append_kernel<D, TURN_ANY><<<grid, AP_NT, 0, st>>>(a);
}

}  // namespace

void launch_rope_table(const double* inv_freq, int pairs, int64_t n, float factor, float2* table, cudaStream_t st) {
  rope_table_kernel<<<(unsigned)ceil_div(n * pairs, 256), 256, 0, st>>>(inv_freq, pairs, n, factor, table);
  count_launch();
}

void launch_kv4_append(const Kv4View& cache, int D, const SeqView& seq, const int32_t* positions, const float2* table,
                       int rot, int interleaved, int64_t max_pos, int q_heads, const HeadRows& q, const HeadRows& k,
                       const HeadRows& v, const HeadRows& q_out, int* err, cudaStream_t st) {
  const int items = q_heads + 2 * cache.kv_heads, per = AP_NT / (D / 8), each = block_tokens(items, per, seq.num_tokens);
  const AppendArgs a{cache, seq, positions, table, rot, interleaved, max_pos, q_heads, q, k, v, q_out, each, err};
  const dim3 grid = token_grid(items, per, seq.num_tokens, each);
  if (D == 128) launch_append<128>(a, grid, st);
  else launch_append<64>(a, grid, st);
  count_launch();
}

void launch_kv4_read(const Kv4View& cache, int D, const SeqView& seq, const HeadRows& k, const HeadRows& v, int* err,
                     cudaStream_t st) {
  const int items = 2 * cache.kv_heads, per = AP_NT / (D / 8), each = block_tokens(items, per, seq.num_tokens);
  const ReadArgs a{cache, seq, k, v, each, err};
  const dim3 grid = token_grid(items, per, seq.num_tokens, each);
  if (D == 128) kv4_read_kernel<128><<<grid, AP_NT, 0, st>>>(a);
  else kv4_read_kernel<64><<<grid, AP_NT, 0, st>>>(a);
  count_launch();
}

}  // namespace kl
