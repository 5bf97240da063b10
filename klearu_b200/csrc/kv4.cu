// kv4.cu -- rotary positions and the paged 4-bit key/value cache: the table of
// angles, appending, reading back.  The layout and the number format are in
// kv4.cuh; attention over the cache is in attend.cu.
//
// klearu-llm's counterpart is its CPU attention half (crates/klearu-llm/src/
// model/kv_cache.rs holds f32 keys and values); the 4-bit pages are this
// engine's own.
#include "engine.h"
#include "kv4.cuh"
#include "pdl.cuh"

namespace kl {
namespace {

// table[p][i] = (cos, sin)(p * inv_freq[i]) * factor, angles and functions in
// 64 bits (a far position's angle has no fraction bits left in 32), held in 32.
__global__ void rope_table_kernel(const double* inv_freq, int pairs, int64_t n, double factor, float2* table) {
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
  if constexpr (MODE == TURN_PAIRS || MODE == TURN_HALVES) {
    if (d0 >= rot) return;
    const float4* p = reinterpret_cast<const float4*>(row + (MODE == TURN_PAIRS ? 4 * l : d0 < half ? d0 : d0 - half));
#pragma unroll
    for (int i = 0; i < (MODE == TURN_PAIRS ? 2 : 4); ++i) *reinterpret_cast<float4*>(&t.cs[2 * i]) = p[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = interleaved ? d0 + 2 * i : d0 + i;
      t.cs[i] = make_float2(1.f, 0.f);
      if ((!interleaved || i < 4) && d < rot) t.cs[i] = row[interleaved ? d >> 1 : d < half ? d : d - half];
    }
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

__device__ __forceinline__ void async_copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

constexpr int AP_NT = 256;
constexpr int AP_RING = 4;     // rows of a thread's ring
constexpr int AP_BLOCKS = 4;   // of an SM
constexpr int AP_EACH = 12;    // most vectors of a group
constexpr int RD_TOKENS = 4;   // most tokens of a block that reads

// Where a token stands: its page and place in it, its position.
struct Place {
  int64_t page;  // -1: nowhere
  int off, pos;
  int kind;  // 0: of no sequence, left as it is; 1: padding or bad, zeros; 2: live
};
// Token t of sequence b.  *bad: something had to be left out.
__device__ __forceinline__ Place find_place(const Kv4View& cache, const SeqView& seq, const int32_t* positions, int b, int t,
                                            bool table, int64_t max_pos, bool* bad) {
  Place r{-1, 0, 0, 0};
  if (b >= seq.num_seqs) return r;
  const SeqSpan s = seq_span(seq, b, cache.page_size, bad);
  if (t < s.row) return r;  // in front of the first sequence
  const int index = s.first + (t - s.row);
  r.pos = positions ? positions[t] : index;
  r.kind = 1;
  if (index < 0) return r;  // in front of its sequence's first token: padding
  if (index < s.kv_len) {
    const int col = kv4_column(cache, index >> 4);
    r.off = index - col * cache.page_size;
    r.page = seq.table[b * seq.table_ld + col];
  }
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

// The places of a block's n tokens from t0 on: its first warp searches the first one's sequence, each lane walks on to
// its own token's, which is hardly ever more than a step away, or searches in what is left.  One chain of loads for all.
__device__ __forceinline__ void find_places(const Kv4View& cache, const SeqView& seq, const int32_t* positions, int t0, int n,
                                            bool table, int64_t max_pos, Place* places, int* err) {
  if (threadIdx.x >= 32) return;
  const int lane = threadIdx.x, t = t0 + min(lane, n - 1), ns = seq.num_seqs;
  int b = find_seq(seq.cu_q, ns, t0);
  for (int i = 0; i < 3 && b < ns && seq.cu_q[b + 1] <= t; ++i) ++b;
  if (b < ns && seq.cu_q[b + 1] <= t) {
    int lo = b + 1, hi = ns;
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (seq.cu_q[mid + 1] <= t) lo = mid + 1;
      else hi = mid;
    }
    b = lo;
  }
  bool bad = false;
  const Place p = find_place(cache, seq, positions, b, t, table, max_pos, &bad);
  if (lane < n) places[lane] = p;
  // sequences of which the call has no row at all
  if (blockIdx.y == 0 && blockIdx.z == 0 && lane == 0 && seq.cu_q[ns] > seq.num_tokens) bad = true;
  if (bad && blockIdx.x == 0) atomicOr(err, DERR_BOUNDS);
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
  int vec;          // all vectors start on 16 bytes
  int shift, each;  // 2^shift groups of lanes take a token of the block, each of them that many of its vectors
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
// The same by a reciprocal: y = d inv, and y + (d - y s) inv, the bracket in one
// fused operation, is the quotient d / s rounded correctly (Markstein, 1990),
// since inv is 1 / s rounded correctly.
__device__ __forceinline__ float quotient(float d, float s, float inv) {
  const float y = d * inv;
  return fmaf(fmaf(-y, s, d), inv, y);
}
__device__ __forceinline__ uint32_t codes8(const float* x, float m, float s) {
  if (!(s > 1e-30f && s < 1e30f)) return exact_codes(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), m, s);
  const float inv = __frcp_rn(s);
  // + 2^23 rounds to a whole number, which stands in the low bits of 0x4b000000 + c
  uint32_t w = 0u, over = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = fminf(fmaxf(quotient(x[i] - m, s, inv), 0.f), 15.f) + 8388608.f;
    w += __float_as_uint(y) << (4 * kv4_nibble(i));
    over += 0x4b000000u << (4 * kv4_nibble(i));
  }
  return w - over;
}

// A group of D / 8 lanes takes the head vectors of one token one by one, 8 dims
// per lane, so that the token's row of the table is loaded once; a block's 16
// (D = 128) or 32 groups are dealt to one or more tokens.  Each thread's 16 bytes
// of a vector come through a ring of its own in shared memory, three vectors
// ahead, which keeps the registers for four blocks an SM.
// 8000 tokens of 32 + 16 heads of 128, half of each turned: 45 us, 3.9 TB/s, with
// three of four issue slots taken: the codes of a key or value cost 250
// instructions a warp, a query 115.  A head vector of several tokens to a group,
// the table rows loaded again for each, was 20% to 35% slower; two tokens in
// registers instead of the ring 15%; quotients on a border taken as divisions 10%.
template <int D, int MODE>
__global__ void __launch_bounds__(AP_NT, AP_BLOCKS) kv4_append_kernel(AppendArgs a) {
  constexpr int L = D / 8;  // lanes of a group
  __shared__ uint4 ring[AP_RING][AP_NT];
  __shared__ Place places[AP_NT / L];
  const int kh = a.cache.kv_heads, items = a.q_heads + 2 * kh;
  const int l = threadIdx.x % L, per = 1 << a.shift, tokens = (AP_NT / L) >> a.shift;
  const int t0 = (int)(((int64_t)blockIdx.z * 65535 + blockIdx.y) * tokens), here = min(tokens, a.seq.num_tokens - t0);
  const int mine = (threadIdx.x / L) >> a.shift, t = t0 + mine;
  const int first = blockIdx.x * per * a.each + (threadIdx.x / L & (per - 1));  // then every per-th: q heads, k, v
  const int n = mine < here && first < items ? min(a.each, (items - first + per - 1) >> a.shift) : 0;
  auto vector_of = [&](int item, int64_t* head, int* end) {  // and its kind's head stride and first item after
    const bool is_q = item < a.q_heads, is_k = item < a.q_heads + kh;
    const HeadRows& in = is_q ? a.q : is_k ? a.k : a.v;
    const int from = is_q ? 0 : is_k ? a.q_heads : a.q_heads + kh;
    *head = in.head;
    *end = is_q ? a.q_heads : from + kh;
    return static_cast<const __nv_bfloat16*>(in.p) + t * in.token + (item - from) * in.head + 8 * l;
  };
  // what is fetched next: its address moves on by a step while the kind stays the same
  int coming = first, kind_end = 0;
  const int stop = first + (n << a.shift);
  int64_t step = 0;
  const __nv_bfloat16* from = nullptr;
  auto fetch = [&](int slot) {  // into a slot that was read a vector ago
    if (coming < stop) {
      if (coming >= kind_end) {
        from = vector_of(coming, &step, &kind_end);
        step <<= a.shift;
      }
      if (a.vec) async_copy16(&ring[slot][threadIdx.x], from);
      else ring[slot][threadIdx.x] = load8_raw(from, false);
      coming += per;
      from += step;
    }
    async_commit();
  };
  begin_next();
  after_before();
#pragma unroll
  for (int i = 0; i < AP_RING - 1; ++i) fetch(i);  // before their places are known
  find_places(a.cache, a.seq, a.positions, t0, here, MODE != TURN_NONE, a.max_pos, places, a.err);
  const unsigned group = (L == 16 ? 0xffffu : 0xffu) << ((threadIdx.x & 31) / L * L);
  __syncthreads();
  if (n == 0) return;
  const Place pl = places[mine];
  const int kind = pl.kind, tok = pl.off & 15;
  __nv_bfloat16* ob = static_cast<__nv_bfloat16*>(a.q_out.p) + t * a.q_out.token + first * a.q_out.head + 8 * l;
  const int64_t out_step = a.q_out.head << a.shift;
  if (kind != 2) {
    async_wait<0>();
    const float none[8] = {};
    if (kind == 1)
      for (int item = first; item < min(stop, a.q_heads); item += per, ob += out_step) store8_bf16(ob, a.q_out.vec, none);
    return;
  }
  unsigned char* tile0 = pl.page < 0 ? nullptr : kv4_tile(a.cache, kv4_tile_bytes(D), pl.page, 0, pl.off >> 4);
  const int k_off = kv4_k_off<D>(tok, l), v_off = kv4_codes(D) + kv4_v_off<D>(tok, l);
  const int head_bytes = a.cache.tiles_per_page * kv4_tile_bytes(D);
  Turn turn;
  if (MODE != TURN_NONE && first < a.q_heads + kh)
    load_turn<MODE>(turn, a.table + (int64_t)pl.pos * (a.rot >> 1), l, a.rot, a.interleaved);

  int slot = 0;
  for (int item = first; item < stop; item += per) {
    fetch((slot + AP_RING - 1) % AP_RING);
    async_wait<AP_RING - 1>();
    const uint4 raw = ring[slot][threadIdx.x];
    slot = (slot + 1) % AP_RING;
    const bool is_q = item < a.q_heads, is_k = !is_q && item < a.q_heads + kh;
    const uint32_t w4[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = __uint_as_float(w4[e] << 16);
      x[2 * e + 1] = __uint_as_float(w4[e] & 0xffff0000u);
    }
    if (MODE != TURN_NONE && (is_q || is_k)) {
      int64_t head;
      int end;
      const __nv_bfloat16* p = MODE == TURN_ANY ? vector_of(item, &head, &end) - 8 * l : nullptr;
      turn8<MODE>(x, turn, p, l, a.rot, a.interleaved, group);
    }
    if (is_q) {
      if (MODE == TURN_ANY) __syncwarp(group);  // q_out may be q: every lane has read its partners
      store8_bf16(ob, a.q_out.vec, x);
      ob += out_step;
      continue;
    }
    if (pl.page < 0) break;  // no place in the cache for this and what follows
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
    const float range = hi - lo;
    __nv_bfloat16 st = __float2bfloat16_rn(range > 1e-30f ? quotient(range, 15.f, 1.f / 15.f) : __fdiv_rn(range, 15.f));
    __nv_bfloat16 mn = __float2bfloat16_rn(lo);
    float sf = to_f(st), mf = to_f(mn);
    if (!fin || !finite_f(sf) || !finite_f(mf)) {
      st = __ushort_as_bfloat16(0);
      mn = __ushort_as_bfloat16(0x7fff);
      sf = 0.f;
    }
    const uint32_t w = sf > 0.f ? codes8(x, mf, sf) : 0u;
    unsigned char* tile = tile0 + (int64_t)(item - a.q_heads - (is_k ? 0 : kh)) * head_bytes;
    *reinterpret_cast<uint32_t*>(tile + (is_k ? k_off : v_off)) = w;
    if (l == 0) {
      const uint32_t pr = (uint32_t)__bfloat16_as_ushort(st) | ((uint32_t)__bfloat16_as_ushort(mn) << 16);
      *reinterpret_cast<uint32_t*>(tile + 2 * kv4_codes(D) + tok * 8 + (is_k ? 0 : 4)) = pr;
    }
  }
  async_wait<0>();  // rows that were not taken
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
  __shared__ Place places[RD_TOKENS];
  const int kh = a.cache.kv_heads;
  const int l = threadIdx.x % L, item = blockIdx.x * PER + threadIdx.x / L;
  const int t0 = (int)(((int64_t)blockIdx.z * 65535 + blockIdx.y) * a.tokens);
  const int n = min(a.tokens, a.seq.num_tokens - t0);
  begin_next();
  after_before();
  find_places(a.cache, a.seq, nullptr, t0, n, false, 0, places, a.err);
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
      const uint32_t even = w[u] & 0x0f0f0f0fu, odd = (w[u] >> 4) & 0x0f0f0f0fu;
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // a byte under 2^23's exponent is that number and a code
        const int n = kv4_nibble(i);
        const uint32_t c = __byte_perm(n & 1 ? odd : even, 0x4b000000u, 0x7540 | (n >> 1));
        x[i] = fmaf(__uint_as_float(c) - 8388608.f, sf, mf);
      }
      store8_bf16(static_cast<__nv_bfloat16*>(o.p) + (int64_t)(t0 + u0 + u) * o.token + head * o.head + 8 * l, o.vec, x);
    }
  }
}

// Reading: four tokens a block where one each would be more blocks than the machine holds at once (8 key heads: 8000
// tokens 10.3 us against 17.6, 600 3.3 both, 256 2.9 against 2.7).
int block_tokens(int items, int per, int tokens) { return ceil_div(items, per) * tokens >= 8 * 148 ? RD_TOKENS : 1; }
dim3 token_grid(int items, int per, int tokens, int each) {
  const int64_t n = ceil_div(tokens, each);
  return dim3((unsigned)ceil_div(items, per), (unsigned)std::min<int64_t>(n, 65535), (unsigned)ceil_div(n, 65535));
}

template <int D>
void launch_append(const AppendArgs& a, dim3 grid, cudaStream_t st) {
  auto* kernel = !a.table ? kv4_append_kernel<D, TURN_NONE>
                 : a.interleaved ? a.rot % 8 == 0 ? kv4_append_kernel<D, TURN_PAIRS> : kv4_append_kernel<D, TURN_ANY>
                 : a.rot % 16 == 0 ? kv4_append_kernel<D, TURN_HALVES> : kv4_append_kernel<D, TURN_ANY>;
  launch_next(kernel, grid, AP_NT, 0, st, a);
}

}  // namespace

void launch_rope_table(const double* inv_freq, int pairs, int64_t n, double factor, float2* table, cudaStream_t st) {
  rope_table_kernel<<<(unsigned)ceil_div(n * pairs, 256), 256, 0, st>>>(inv_freq, pairs, n, factor, table);
  count_launch();
}

void launch_kv4_append(const Kv4View& cache, int D, const SeqView& seq, const int32_t* positions, const float2* table,
                       int rot, int interleaved, int64_t max_pos, int q_heads, const HeadRows& q, const HeadRows& k,
                       const HeadRows& v, const HeadRows& q_out, int* err, cudaStream_t st) {
  // One vector a group while that gives each processor two blocks at most, up to AP_EACH for more.  48 heads of 128:
  // 64 tokens and reading them back take 8.3 us with one or four each and 10.4 with eight, 500 tokens 14.2, 10.4 and
  // 12.5, 8000 tokens 108, 74 and 66 and with twelve 63.
  const int items = q_heads + 2 * cache.kv_heads, groups = AP_NT / (D / 8);
  const int64_t turns = (int64_t)items * seq.num_tokens / ((int64_t)groups * 2 * 148);
  const int each = (int)std::min<int64_t>(AP_EACH, std::max<int64_t>(1, turns));
  int shift = 0;
  while ((1 << shift) < groups && (each << shift) < items) ++shift;
  const AppendArgs a{cache, seq, positions, table, rot, interleaved, max_pos, q_heads, q, k, v, q_out,
                     (q_heads == 0 || q.vec) && k.vec && v.vec, shift, each, err};
  const dim3 grid = token_grid(items, each << shift, seq.num_tokens, groups >> shift);
  if (D == 128) launch_append<128>(a, grid, st);
  else launch_append<64>(a, grid, st);
  count_launch();
}

void launch_kv4_read(const Kv4View& cache, int D, const SeqView& seq, const HeadRows& k, const HeadRows& v, int* err,
                     cudaStream_t st) {
  const int items = 2 * cache.kv_heads, per = AP_NT / (D / 8), each = block_tokens(items, per, seq.num_tokens);
  const ReadArgs a{cache, seq, k, v, each, err};
  const dim3 grid = token_grid(items, per, seq.num_tokens, each);
  launch_next(D == 128 ? kv4_read_kernel<128> : kv4_read_kernel<64>, grid, AP_NT, 0, st, a);
  count_launch();
}

}  // namespace kl
