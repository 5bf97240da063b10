// attend_tc.cu -- attention over the paged 4-bit cache for many rows (prompt
// chunks), on tcgen05.  Definitions are in attend.cu.
//
// One block takes 256 rows (token, query head) of one key head as two tiles of
// 128, so that one tile multiplies while the other takes its softmax:
//  * warps 0-3 and 4-7: softmax of tile 0 and 1, one row per thread, 64 scores
//    in registers at a time; P goes back to tensor memory as f16, over the
//    scores that it came from; O is rescaled in place only when a row's maximum
//    has risen by more than 2^8;
//  * warps 8-11: the next 128 keys and values, codes read from global memory
//    one step ahead, turned into f16 (s c + m in one rounding) and written to
//    shared memory in the tensor core's swizzled layouts, K with D contiguous,
//    V as it stands (its tokens are the product's K, "MN-major");
//  * a thread of warp 12: the products, O_i += P_i . V and then S_i = Q_i . K^T
//    of the next step, the tiles in turn, which keeps their softmaxes apart.
//    Few barriers (a commit each) and rolled loops: the four roles share the
//    instruction caches, and unrolling this one over the tiles cost 14%.
// f16, not bf16, for its 11 bits: with keys, values and probabilities at 2^-12
// the output is as exact as its own bf16 rounding.  Its range is made up for by
// powers of two: of each row of Q, of each step's K (both into the score's
// factor) and V.  V is held times 2^-ev, a row's O in units of 2^(unit - 6) of
// its own, and P is 2^(6 + ev - unit) times the probability (to the reference),
// 2^15 at most and with full precision down to 2^-14: the unit follows ev where
// it falls by more than 7, and rises where P would not fit (O is rescaled with
// it), so that neither zeros nor larger values in front leave later probabilities
// among f16's subnormals, and large values count by their probabilities.  A step
// whose keys or values are more than 2^12 apart in size is "wide": there every
// token has powers of two of its own, and each row takes its scores and its unit
// from the tokens that it sees, so that those that it does not see cost it no
// bits; tokens that no row of the block sees are zeros.
// Tensor memory: S_0, S_1 (128 columns each), O_0, O_1 (D columns each).
// Where the rows make fewer blocks than the device has processors (a chunk of
// one long prompt), each row's steps are shared out to several blocks, whose
// averages and sums attend_join_kernel brings together: 64 new tokens of a
// sequence of 60000, 8 key heads: 1122 us in one share, 93 in 18.
//
// 7416 prompt tokens of up to 6000, 32 heads on 8 of 128: 506 us, 692 TFLOP/s.
// Per 128 keys and 256 rows the tensor cores need 2048 cycles and the 32768
// exponentials as many of the special function units; a step takes about 5000
// (tensor cores 37% busy, 1.94 of 4 issue slots, logic 41%): no unit is at its
// limit.  P lies over the scores that it came from, so a tile's next scores wait
// for its whole P . V, whose commit and the next Q . K^T lie between two of its
// softmaxes, while decoding warps share the softmax warps' schedulers.
// Tried without gain: two threads to a row (twice the softmax warps), a quarter
// of the exponentials as polynomials, scores of 64 keys (a product reads all of
// Q whatever its width), P and its product in halves.
#include <cuda_fp16.h>

#include <cstddef>

#include "attend.cuh"
#include "engine.h"
#include "tcgen05.cuh"

namespace kl {
namespace {

constexpr int TC_KV = 128;   // keys per step
constexpr int TC_ROWS = 256;  // rows per block
constexpr int TC_NT = 512;    // 4 warpgroups

// MN-major operand, 128-byte swizzle: 64 values of N in 128 bytes, 8 of K in
// 1024; the next 64 of N are lbo bytes on, the next 8 of K 1024.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// A from tensor memory (f16, two values of K per column)
__device__ __forceinline__ void tc5_mma_ta(uint32_t tmem, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem),
      "r"(ta), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}
#define TC_R32(v) \
  "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), \
      "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), \
      "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), \
      "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
__device__ __forceinline__ void tc5_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : TC_R32(v)
      : "r"(taddr));
}
#undef TC_R32
__device__ __forceinline__ void tc5_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};\n" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tc5_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// codes in nibbles 0 and 4 of w as f16 s c + m, one rounding
__device__ __forceinline__ uint32_t value2(uint32_t w, uint32_t s2, uint32_t m2) {
  const uint32_t v = (w & 0x000f000fu) | 0x64006400u;  // 1024 + c, exact
  uint32_t c, r;
  asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(c) : "r"(v), "r"(0x64006400u));
  asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(r) : "r"(c), "r"(s2), "r"(m2));
  return r;
}
// the 8 dims of a word as 16 bytes
__device__ __forceinline__ uint4 values8(uint32_t w, uint32_t s2, uint32_t m2) {
  return make_uint4(value2(w, s2, m2), value2(w >> 4, s2, m2), value2(w >> 8, s2, m2), value2(w >> 12, s2, m2));
}
__device__ __forceinline__ uint32_t twice_f16(float x) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %1;\n" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float bf_low(uint32_t pr) { return __uint_as_float(pr << 16); }           // a step
__device__ __forceinline__ float bf_high(uint32_t pr) { return __uint_as_float(pr & 0xffff0000u); }  // a minimum
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127
// what a vector's values do not pass; zero where its minimum is NaN
__device__ __forceinline__ uint32_t reach(uint32_t pr) {
  const float s = bf_low(pr), m = bf_high(pr);
  return m == m ? __float_as_uint(fmaxf(fabsf(m), fabsf(fmaf(15.f, s, m)))) : 0u;
}
// two f32 operations an instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int D>
struct TcSmem {
  static constexpr int Q = 128 * D * 2;     // one tile
  static constexpr int KV = TC_KV * D * 2;  // one stage of K or V
  static constexpr int BYTES = 2 * Q + 4 * KV + 1024;
};

// A step's powers of two and missing pages.
struct TcStep {
  unsigned char hole[8];  // 16-token tiles whose page does not exist
  float ek2;              // K is held times 1 / ek2; negative: a wide step
  float ev;               // V times 2^-ev; TC_NONE: nothing but zeros
};
// Of a token: K is held times 2^-ek, V times 2^-ev, of the whole step alike where it is not wide.
struct TcPowers {
  signed char ek, ev;  // ev -128: its value is zero
};
// Of a step that is not wide, as a power of two: P has steps of 2^-24 and is at least 2^-1 times the probability, so that a
// value 2^12 larger than those that count errs by 2^-12 of them, as f16 does.
constexpr int TC_SPREAD = 12;
constexpr float TC_NONE = -10000.f;
struct TcShared {
  uint64_t q_full, k_full[2], v_full[2], done;
  uint64_t s_full[2], p_full[2], o_full[2];  // by tile, one phase a step: scores there; P there; O has taken P
  uint32_t tmem;
  int fail;
  alignas(16) uint32_t reach[2][4][4];  // by step & 1: largest |K|, |V|, smallest of each but 0, of each decoding warp
  // by step & 3: a step's is written again when the step two on has its scores, after this one's softmax
  alignas(16) TcStep step[4];
  alignas(16) TcPowers powers[4][TC_KV];
};
static_assert(offsetof(TcShared, reach) % 16 == 0 && offsetof(TcShared, step) % 16 == 0 && sizeof(TcStep) == 16,
              "read as 16- and 8-byte vectors");
// every lane's answer, so that a warp gives up as one
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(FULL, mbar_wait(bar, parity));
}

// the decoding warps' barrier, and whether all of their threads said yes
__device__ __forceinline__ bool all_of_128(bool yes) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.pred.aligned q, 1, 128, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)yes)
      : "memory");
  return r != 0;
}

// One pair of row tiles of one sequence, or its share of one chunk of the keys.
struct TcWork {
  SeqSpan s;
  int b, rows, r0, first;  // row r is token first + r / group
  int lo, steps;           // keys [lo, lo + 128 steps) cover what the rows see (there); lo a multiple of 16
  int from;                // no row sees a key in front of it
  int hi;                  // no row sees hi or later (the chunk ends there)
};

// Calls f(work) for each of this block's pairs of tiles until it returns false.
// The last rows of a sequence see most: they go first.
template <class F>
__device__ __forceinline__ void tc_each(const AttendArgs& a, int chunks, TcShared& sh, bool* bad, F f) {
  const int group = a.q_heads / a.cache.kv_heads;
  const int height = (int)gridDim.x / chunks, chunk = (int)blockIdx.x / height;
  TcWork w;
  for (w.b = blockIdx.z; w.b < a.seq.num_seqs; w.b += gridDim.z) {
    w.s = seq_span(a.seq, w.b, a.cache.page_size, bad);
    w.rows = w.s.q_len * group;
    w.first = w.s.first;
    const int tiles = (w.rows + TC_ROWS - 1) / TC_ROWS;
    for (int rt = height - 1 - ((int)blockIdx.x - chunk * height); rt < tiles; rt += height) {
      w.r0 = rt * TC_ROWS;
      const int pos0 = w.first + w.r0 / group;
      w.hi = min(w.first + (min(w.r0 + TC_ROWS, w.rows) - 1) / group + 1, w.s.kv_len);
      w.from = window_from(a.window, pos0);
      w.lo = w.from & ~15;
      w.steps = w.hi > w.lo ? (w.hi - w.lo + TC_KV - 1) / TC_KV : 0;
      if (chunks > 1) {  // the rows' own steps in equal shares
        const int each = (w.steps + chunks - 1) / chunks, from = min(w.steps, chunk * each);
        w.steps = min(w.steps - from, each);
        w.lo += from * TC_KV;
        w.hi = min(w.hi, w.lo + w.steps * TC_KV);
      }
      if (!f(w)) {  // a wait gave up
        sh.fail = 1;
        return;
      }
    }
  }
}

// What a row's softmax has so far.
struct TcRow {
  float ref, lift, l;  // l: the sum of 2^(score - ref); a score above lift moves ref
  float unit, peak;    // of O; the largest so far: O stays finite while the unit is above peak - 64
};
// A wide step's probabilities, for a row that sees its keys [from, to].  Not inlined: beside the ordinary step's its code
// costs that one 16 us of 507 (7416 prompt tokens).
template <int D>
__device__ __noinline__ TcRow tc_wide_step(TcRow row, const TcStep& st, const TcPowers* powers, float worth, int from, int to,
                                           uint32_t tS, uint32_t tO, bool rescale) {
  // 16 keys' scores in units of log2, -inf for those that it does not see, and their values' powers
  auto scores = [&](int c, float* t, float* ev) {
    uint32_t s[16];
    tc5_ld16_async(tS + c, s);
    const uint4 x[2] = {*reinterpret_cast<const uint4*>(powers + c), *reinterpret_cast<const uint4*>(powers + c + 8)};
    const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
    const bool hole = st.hole[c >> 4];
    tc5_ld_wait();
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const uint32_t y = w[u >> 1] >> (16 * (u & 1));
      const float f = fminf(fmaxf(worth * pow2((signed char)(y & 0xff)), 1.2e-38f), 3.4e38f);
      t[u] = c + u <= to && c + u >= from && !hole ? __uint_as_float(s[u]) * f : -INFINITY;
      ev[u] = __int_as_float(0x4b400000 + (signed char)(y >> 8 & 0xff)) - 12582912.f;
    }
  };
  // the largest score, and the largest with its value's exponent, that one relative to the first: scores may be large
  float top = -INFINITY, most = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < TC_KV; c += 16) {
    float t[16], ev[16];
    scores(c, t, ev);
    float now = top;
#pragma unroll
    for (int u = 0; u < 16; ++u) now = fmaxf(now, t[u]);
    if (now > top) most -= now - top;
    top = now;
#pragma unroll
    for (int u = 0; u < 16; ++u)
      if (ev[u] != -128.f && t[u] != -INFINITY) most = fmaxf(most, t[u] - top + ev[u]);
  }
  float by = 1.f;  // of O
  const bool first = row.lift == -INFINITY;
  if (top != -INFINITY && (first || top > row.ref)) {
    if (!first) by = exp2_fast(row.ref - top);
    row.ref = top;
    row.lift = top + 8.f;
    row.l *= by;
  }
  if (most != -INFINITY) {  // the unit by what counts most
    float need = ceilf(fminf(fmaxf(most + (top - row.ref), -126.f), 126.f));
    if (row.unit == TC_NONE || first) {
      row.unit = need;
    } else {
      need = fmaxf(need, row.peak - 64.f);
      if (need > row.unit + 1.f || need < row.unit - 7.f) {
        by *= pow2(max(-126, (int)(row.unit - need)));
        row.unit = need;
      }
    }
    row.peak = fmaxf(row.peak, row.unit);
  }
  if (rescale && __any_sync(FULL, by != 1.f)) {
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
      uint32_t v[16];
      tc5_ld16_async(tO + c, v);
      tc5_ld_wait();
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u] = __float_as_uint(__uint_as_float(v[u]) * by);
      tc5_st16(tO + c, v);
    }
  }
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < TC_KV; c += 32) {  // P's columns [c / 2, c / 2 + 16) have been read
    uint32_t pk[16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float t[16], ev[16];
      scores(c + 16 * h, t, ev);
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        sum += exp2_fast(t[u] - row.ref);
        t[u] = exp2_fast(t[u] - row.ref + (ev[u] == -128.f ? 0.f : 6.f + ev[u] - row.unit));
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) pk[8 * h + u] = pack_f16(t[2 * u], t[2 * u + 1]);
    }
    tc5_st16(tS + c / 2, pk);
  }
  row.l += sum;
  tc5_st_wait();
  return row;
}

// ---- warps 0-7: one row per thread ----
template <int D>
__device__ __forceinline__ void tc_softmax(const AttendArgs& a, int chunks, TcShared& sh, unsigned char* sQ, bool* bad) {
  constexpr int LPR = D / 8, RPI = 32 / LPR;  // a row's lanes where a warp moves rows, 16 bytes each; rows at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = warp >> 2, r = threadIdx.x & 127;
  const int kvh = blockIdx.y, group = a.q_heads / a.cache.kv_heads;
  const uint32_t lane_off = (uint32_t)(warp & 3) << 21;
  const uint32_t tS = sh.tmem + i * 128 + lane_off, tO = sh.tmem + 256 + i * D + lane_off;
  // row x, chunk c of 16 bytes of this tile's share of shared memory: the 128-byte swizzle
  unsigned char* tile = sQ + i * TcSmem<D>::Q;
  auto place = [&](int x, int c) {
    return reinterpret_cast<uint4*>(tile + (c >> 3) * 16384 + x * 128 + (((c & 7) ^ (x & 7)) << 4));
  };
  const int sub = lane / LPR, chunk = lane % LPR, warp_row = r & ~31;
  uint32_t kq = 0;
  tc_each(a, chunks, sh, bad, [&](const TcWork& w) {
    const int row = w.r0 + i * 128 + r;
    const int rows_here = w.rows - (w.r0 + i * 128 + warp_row);  // of this warp's 32, how many there are
    float worth = 0.f;  // of a score, in units of log2, but for the keys' power of two
    if (w.steps > 0) {
      // the rows of Q as f16, each with its largest value in [2^13, 2^14), K-major; a row by LPR lanes
      const int64_t mine = (w.s.row + row / group) * a.q.token + (kvh * group + row % group) * a.q.head;
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q.p) + 8 * chunk;
      const float factor = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 raw[LPR / 2];  // their loads at once: nothing else runs until the first scores
#pragma unroll
        for (int u = 0; u < LPR / 2; ++u) {
          const int x = (h * (LPR / 2) + u) * RPI + sub;
          const int64_t at = __shfl_sync(FULL, mine, x);
          raw[u] = x < rows_here ? load8_raw(q + at, a.q.vec) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < LPR / 2; ++u) {
          const int x = (h * (LPR / 2) + u) * RPI + sub;
          uint32_t v[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w}, top = 0;  // the largest |x|, as bf16 bits
#pragma unroll
          for (int e = 0; e < 4; ++e) top = __vmaxu2(top, v[e] & 0x7fff7fffu);
          top = max(top & 0xffffu, top >> 16);
#pragma unroll
          for (int d = 1; d < LPR; d <<= 1) top = max(top, __shfl_xor_sync(FULL, top, d));
          const int eq = top < 0x7f80u ? max(-114, min(100, 13 - ((int)(top >> 7) - 127))) : 0;
          // the scale's sign goes into q, and a scale of zero makes it zero, so that a score's factor is positive
          const float up = a.scale == 0.f ? 0.f : a.scale < 0.f ? -pow2(eq) : pow2(eq);
#pragma unroll
          for (int e = 0; e < 4; ++e)  // a row that is not finite is NaN
            v[e] = top < 0x7f80u ? pack_f16(__uint_as_float(v[e] << 16) * up, __uint_as_float(v[e] & 0xffff0000u) * up)
                                 : 0x7fff7fffu;
          *place(warp_row + x, chunk) = make_uint4(v[0], v[1], v[2], v[3]);
          const float its = __shfl_sync(FULL, factor * pow2(-eq), (lane % RPI) * LPR);
          if (lane / RPI == h * (LPR / 2) + u) worth = its;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full);
    }
    const int own = w.first + row / group - w.lo, seen = min(own, w.s.kv_len - 1 - w.lo);  // counted from w.lo, as what follows
    // every row of the tile sees all of the steps in (jlo, jhi)
    const int jhi = (min(w.first + (w.r0 + i * 128) / group, w.s.kv_len - 1) - w.lo + 1) / TC_KV;
    const int last = w.first + (min(w.r0 + i * 128 + 128, w.rows) - 1) / group - w.lo;
    const int jlo = a.window > 0 && last >= a.window ? (last - a.window + TC_KV) / TC_KV - 1 : -1;
    float ref = 0.f, lift = -INFINITY, l = 0.f, unit = TC_NONE, peak = -126.f;  // a TcRow
    const float most_worth = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(worth)));
    for (int j = 0; j < w.steps; ++j) {
      if (!warp_wait(&sh.s_full[i], (kq + j) & 1u)) return false;
      tc5_fence_after();
      const TcStep& st = sh.step[(kq + j) & 3u];
      const uint2 holes = *reinterpret_cast<const uint2*>(st.hole);
      // .. or scores that may pass 2^22, where the ordinary step's one rounding of a score and its reference would differ
      if (st.ek2 < 0.f || most_worth * st.ek2 > 0x1p-13f) {
        const int to = seen - TC_KV * j, from = window_from(a.window, own - TC_KV * j);
        const TcRow row = tc_wide_step<D>({ref, lift, l, unit, peak}, st, sh.powers[(kq + j) & 3u], worth, from, to, tS, tO, j > 0);
        ref = row.ref, lift = row.lift, l = row.l, unit = row.unit, peak = row.peak;
        tc5_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[i]);
        continue;
      }
      float off = st.ev - unit;  // P is 2^(6 + off) times the probability
      float grow = 1.f;          // of O by a fall of its unit
      if (!(off >= -7.f && off < 1000.f) || lift == -INFINITY) {
        if (unit != TC_NONE && st.ev != TC_NONE && lift != -INFINITY) grow = pow2((int)-off);  // else O is zero, or stays
        if (st.ev != TC_NONE) unit = st.ev, peak = fmaxf(peak, unit);
        off = 0.f;
      }
      const float f = fmaxf(worth * st.ek2, 1.2e-38f);  // never 0, which an unseen score's -inf would make NaN
      uint64_t sum2[4] = {0, 0, 0, 0};
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {  // 64 scores at a time, which fit the registers
        float s[64];
        tc5_ld32(tS + 64 * h, reinterpret_cast<uint32_t*>(s));
        tc5_ld32(tS + 64 * h + 32, reinterpret_cast<uint32_t*>(s) + 32);
        tc5_ld_wait();
        const uint32_t hole4 = h ? holes.y : holes.x;
        if (j >= jhi || j <= jlo) {
          const int at0 = TC_KV * j + 64 * h, to = seen - at0, from = window_from(a.window, own - at0);  // columns seen
          const unsigned span = to >= from ? (unsigned)(to - from) : 0u, at = to >= from ? (unsigned)from : 0x40000000u;
#pragma unroll
          for (int u = 0; u < 64; ++u)
            if ((unsigned)u - at > span) s[u] = -INFINITY;
        }
        if (hole4) {
#pragma unroll
          for (int u = 0; u < 64; ++u)
            if (hole4 >> (8 * (u >> 4)) & 1u) s[u] = -INFINITY;
        }
        // maxima and sums in four chains: a warp has its scheduler almost to itself, so latency counts
        float tops[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) tops[u] = fmaxf(s[u], s[u + 4]);
#pragma unroll
        for (int u = 8; u < 64; u += 8)
#pragma unroll
          for (int c = 0; c < 4; ++c) tops[c] = fmaxf(tops[c], fmaxf(s[u + c], s[u + c + 4]));
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        if (top != -INFINITY) top *= f;
        if (__any_sync(FULL, top > fminf(lift, lift + 1.f - off) || grow != 1.f)) {
          const bool first = lift == -INFINITY;
          const float now = top > lift - 8.f || first ? top : ref;
          float keep = 1.f;
          if (now != -INFINITY) {
            keep = first ? 1.f : exp2_fast(ref - now);
            ref = now;
            lift = now + 8.f;
          }
          l *= keep;
          // larger values than the unit's keep it as long as their keys' scores are as much lower
          const float room = floorf(ref - top);
          if (off > room + 1.f) {
            keep *= pow2(max(-126, (int)(room - off)));
            unit += off - room;
            peak = fmaxf(peak, unit);
            off = room;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) sum2[c] = mul2(sum2[c], pair(keep, keep));
          if (h == 1) {  // the step's first probabilities
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              uint32_t v[16];
              tc5_ld16_async(tS + 16 * c, v);
              tc5_ld_wait();
#pragma unroll
              for (int u = 0; u < 16; ++u) {
                const __half2 p = *reinterpret_cast<__half2*>(&v[u]);
                v[u] = pack_f16(__low2float(p) * keep, __high2float(p) * keep);
              }
              tc5_st16(tS + 16 * c, v);
            }
          }
          if (j > 0) {  // O: these scores were not begun before it had taken the step before
            const float by = keep * grow;
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t v[16];
              tc5_ld16_async(tO + 16 * c, v);
              tc5_ld_wait();
#pragma unroll
              for (int u = 0; u < 16; ++u) v[u] = __float_as_uint(__uint_as_float(v[u]) * by);
              tc5_st16(tO + 16 * c, v);
            }
          }
          grow = 1.f;
        }
        const uint64_t f2 = pair(f, f), less2 = pair(6.f + off - ref, 6.f + off - ref);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            uint64_t v = fma2(pair(s[32 * c + 2 * u], s[32 * c + 2 * u + 1]), f2, less2);
            float x, y;
            unpair(v, x, y);
            x = exp2_fast(x);
            y = exp2_fast(y);
            sum2[u & 3] = add2(sum2[u & 3], pair(x, y));
            pk[u] = pack_f16(x, y);
          }
          tc5_st16(tS + 32 * h + 16 * c, pk);
        }
        if (h == 0) tc5_st_wait();  // the second half may read them back
      }
      float x, y;
      unpair(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), x, y);
      l = fmaf(x + y, off == 0.f ? 0.015625f : exp2f(-6.f - off), l);
      tc5_st_wait();
      tc5_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[i]);
    }
    if (chunks > 1) {  // for the join: the rows' averages with log2 of their sums, no row where nothing was seen
      const int64_t at = ((int64_t)((int)blockIdx.x / ((int)gridDim.x / chunks)) * a.seq.num_tokens + w.s.row + row / group) *
                             a.q_heads + kvh * group + row % group;
      const bool mine = row < w.rows;
      if (mine) reinterpret_cast<float2*>(a.scratch)[at] = l == 0.f ? make_float2(-INFINITY, 0.f) : make_float2(ref + log2f(l), 1.f);
      if (w.steps == 0) return true;
      kq += (uint32_t)w.steps;
      if (!warp_wait(&sh.o_full[i], (kq - 1) & 1u)) return false;
      tc5_fence_after();
      const float inv = 0.015625f / l, up = unit == TC_NONE ? 0.f : pow2((int)unit);
      float* to = join_rows(a, chunks) + at * D;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        tc5_ld32(tO + 32 * c, v);
        tc5_ld_wait();
        if (mine && l != 0.f)
#pragma unroll
          for (int u = 0; u < 32; u += 4)
            *reinterpret_cast<float4*>(to + 32 * c + u) =
                make_float4(__uint_as_float(v[u]) * inv * up, __uint_as_float(v[u + 1]) * inv * up,
                            __uint_as_float(v[u + 2]) * inv * up, __uint_as_float(v[u + 3]) * inv * up);
      }
      tc5_fence_before();  // the next rows' first product overwrites O
      __syncwarp();
      return true;
    }
    // O through the rows' place in shared memory, whose queries are done with, so that a row is stored by LPR lanes
    if (w.steps > 0) {
      kq += (uint32_t)w.steps;
      if (!warp_wait(&sh.o_full[i], (kq - 1) & 1u)) return false;
      tc5_fence_after();
      const float inv = l == 0.f ? 0.f : 0.015625f / l, up = unit == TC_NONE ? 0.f : pow2((int)unit);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        tc5_ld32(tO + 32 * c, v);
        tc5_ld_wait();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            y[e] = l == 0.f ? 0u
                            : pack_bf16(__uint_as_float(v[8 * u + 2 * e]) * inv * up,
                                        __uint_as_float(v[8 * u + 2 * e + 1]) * inv * up);
          *place(r, 4 * c + u) = make_uint4(y[0], y[1], y[2], y[3]);
        }
      }
      tc5_fence_before();  // the next rows' first product overwrites O
    } else {
      for (int c = 0; c < LPR; ++c) *place(r, c) = make_uint4(0, 0, 0, 0);
    }
    __syncwarp();
    const int64_t mine = (w.s.row + row / group) * a.out.token + (kvh * group + row % group) * a.out.head;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out.p) + 8 * chunk;
#pragma unroll 4
    for (int u = 0; u < LPR; ++u) {
      const int x = u * RPI + sub;
      const int64_t at = __shfl_sync(FULL, mine, x);
      if (x < rows_here) store8_raw(out + at, a.out.vec, *place(warp_row + x, chunk));
    }
    __syncwarp();
    return true;
  });
}

// ---- warps 8-11: keys and values ----
template <int D>
__device__ __forceinline__ void tc_decode(const AttendArgs& a, int chunks, TcShared& sh, unsigned char* sK, unsigned char* sV,
                                          bool* bad) {
  constexpr int TB = kv4_tile_bytes(D), CODES = kv4_codes(D), KVB = TcSmem<D>::KV;
  const int lane = threadIdx.x & 31, tid = threadIdx.x - 256, sub = tid & 15;
  const int kvh = blockIdx.y;
  uint32_t kq = 0;
  bool alive = true;
  tc_each(a, chunks, sh, bad, [&](const TcWork& w) {
    int ev_top = -126;
    const int32_t* table = a.seq.table + w.b * a.seq.table_ld;
    uint4 kc[D / 32], vc[D / 32], vp[2];
    uint2 kp;
    auto page_of = [&](int j) {
      const int n = w.lo + j * TC_KV + (tid & ~15);
      return j < w.steps && n < w.hi ? table[kv4_column(a.cache, n >> 4)] : -1;
    };
    auto is_hole = [&](int j, int32_t page) {
      return j < w.steps && w.lo + j * TC_KV + (tid & ~15) < w.hi && (page < 0 || page >= a.cache.num_pages);
    };
    // this thread's 16-token tile of step j, null where there is none
    auto tile_of = [&](int j, int32_t page) -> const unsigned char* {
      const int n = (w.lo + j * TC_KV + (tid & ~15)) >> 4;
      return page < 0 || page >= a.cache.num_pages
                 ? nullptr
                 : kv4_tile(a.cache, TB, page, kvh, n - kv4_column(a.cache, n) * a.cache.tiles_per_page);
    };
    // tokens that no row sees are zeros, whatever is left in their places
    auto live = [&](int n) { return n >= w.from && n < w.hi; };
    auto fetch_k = [&](const unsigned char* tile, int j) {
      kp = make_uint2(0, 0);
      if (!tile) {
#pragma unroll
        for (int u = 0; u < D / 32; ++u) kc[u] = make_uint4(0, 0, 0, 0);
        return;
      }
      if (live(w.lo + j * TC_KV + tid)) kp = *reinterpret_cast<const uint2*>(tile + 2 * CODES + sub * 8);
#pragma unroll
      for (int u = 0; u < D / 32; ++u) {
        if (D == 128) {
          kc[u] = *reinterpret_cast<const uint4*>(tile + sub * 64 + u * 16);
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(tile + (sub & 7) * 64 + 2 * u * 16 + (sub >> 3) * 8);
          const uint2 y = *reinterpret_cast<const uint2*>(tile + (sub & 7) * 64 + (2 * u + 1) * 16 + (sub >> 3) * 8);
          kc[u] = make_uint4(x.x, x.y, y.x, y.y);
        }
      }
    };
    auto fetch_v = [&](const unsigned char* tile, int j) {
      if (!tile) {
#pragma unroll
        for (int u = 0; u < D / 32; ++u) vc[u] = make_uint4(0, 0, 0, 0);
        vp[0] = vp[1] = make_uint4(0, 0, 0, 0);
        return;
      }
#pragma unroll
      for (int u = 0; u < D / 32; ++u) vc[u] = *reinterpret_cast<const uint4*>(tile + CODES + (sub + 16 * u) * 16);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        vp[h] = *reinterpret_cast<const uint4*>(tile + 2 * CODES + (8 * h + 2 * (sub & 3)) * 8);
      const int n = w.lo + j * TC_KV;
      if (!live(n) || !live(n + TC_KV - 1)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int m = n + (tid & ~15) + 8 * h + 2 * (sub & 3);
          if (!live(m)) vp[h].x = vp[h].y = 0;
          if (!live(m + 1)) vp[h].z = vp[h].w = 0;
        }
      }
    };
    int32_t page = page_of(0), next = page_of(1);
    const unsigned char* tile = tile_of(0, page);
    fetch_k(tile, 0);
    fetch_v(tile, 0);
    for (int j = 0; j < w.steps; ++j) {
      const uint32_t q = kq + j, st = q & 1u;
      // ---- the step's powers of two: the largest |K| and |V| to [2^13, 2^14) ----
      // a vector that is not finite: the key becomes NaN for whoever sees it, the value zero, since a
      // product with it reaches rows that do not
      const bool nan = bf_high(kp.x) != bf_high(kp.x) || bf_high(kp.y) != bf_high(kp.y);
      const uint32_t my_k = nan ? 0u : reach(kp.x), my_v = nan ? 0u : reach(kp.y);
      const uint32_t rk = __reduce_max_sync(FULL, my_k), rv = __reduce_max_sync(FULL, my_v);
      const uint32_t nk = __reduce_min_sync(FULL, my_k ? my_k : ~0u), nv = __reduce_min_sync(FULL, my_v ? my_v : ~0u);
      if (lane == 0) {
        sh.reach[st][0][tid >> 5] = rk;
        sh.reach[st][1][tid >> 5] = rv;
        sh.reach[st][2][tid >> 5] = nk;
        sh.reach[st][3][tid >> 5] = nv;
      }
      // tile 1's scores of the step before are there: K's and V's stages of two steps before are free (its O had
      // taken P before them), and so is the step's slot.  The four warps give up as one.
      if (q >= 1 && alive) alive = warp_wait(&sh.s_full[1], (q - 1) & 1u);
      const bool hole = is_hole(j, page);
      if (hole) *bad = true;
      if (alive && sub == 0) sh.step[q & 3u].hole[tid >> 4] = hole;
      if (!all_of_128(alive)) return false;
      const uint4 mk = *reinterpret_cast<const uint4*>(sh.reach[st][0]);
      const uint4 mv = *reinterpret_cast<const uint4*>(sh.reach[st][1]);
      const uint4 sk = *reinterpret_cast<const uint4*>(sh.reach[st][2]);
      const uint4 sv = *reinterpret_cast<const uint4*>(sh.reach[st][3]);
      const uint32_t tk = max(max(mk.x, mk.y), max(mk.z, mk.w)), tv = max(max(mv.x, mv.y), max(mv.z, mv.w));
      const uint32_t bk = min(min(sk.x, sk.y), min(sk.z, sk.w)), bv = min(min(sv.x, sv.y), min(sv.z, sv.w));
      auto power = [](uint32_t r) { return max(-126, (int)(r >> 23) - 127 - 13); };  // -126 for 0
      const int ek = power(tk), ev = power(tv);
      // also where values fall so far below those before that the rows' units could not follow
      const bool wide = (tk >> 23) > (bk >> 23) + TC_SPREAD || (tv >> 23) > (bv >> 23) + TC_SPREAD || (tv && ev < ev_top - 60);
      ev_top = max(ev_top, ev);
      sh.powers[q & 3u][tid] = wide ? TcPowers{(signed char)power(my_k), (signed char)(my_v ? power(my_v) : -128)}
                                    : TcPowers{(signed char)ek, (signed char)(tv ? ev : -128)};
      if (tid == 0) {
        sh.step[q & 3u].ek2 = wide ? -1.f : pow2(ek);
        sh.step[q & 3u].ev = tv ? (float)ev : TC_NONE;
      }
      const float fk = pow2(wide ? -power(my_k) : -ek), fv = pow2(-ev);
      {  // ---- K: this thread's token, D contiguous ----
        const uint32_t s2 = nan ? 0u : twice_f16(bf_low(kp.x) * fk);
        const uint32_t m2 = nan ? 0x7fff7fffu : twice_f16(bf_high(kp.x) * fk);
        unsigned char* to = sK + st * KVB + tid * 128;
#pragma unroll
        for (int u = 0; u < D / 8; ++u) {
          const uint4& k = kc[u >> 2];
          const uint32_t word = (u & 3) == 0 ? k.x : (u & 3) == 1 ? k.y : (u & 3) == 2 ? k.z : k.w;
          *reinterpret_cast<uint4*>(to + (u >> 3) * 16384 + (((u & 7) ^ (tid & 7)) << 4)) = values8(word, s2, m2);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.k_full[st]);
      // the next step's loads go out as soon as their registers are free
      page = next;
      tile = tile_of(j + 1, page);
      fetch_k(tile, j + 1);
      next = page_of(j + 2);
      // ---- V: 16-byte chunks of the codes; two tokens each ----
      uint32_t s2[2][2], m2[2][2];  // of tokens 2t + o of half h
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const uint32_t k = o ? vp[h].z : vp[h].x, v = o ? vp[h].w : vp[h].y;
          const bool nan = bf_high(k) != bf_high(k) || bf_high(v) != bf_high(v);
          const float fo = wide ? pow2(-power(reach(v))) : fv;
          s2[h][o] = nan ? 0u : twice_f16(bf_low(v) * fo);
          m2[h][o] = nan ? 0u : twice_f16(bf_high(v) * fo);
        }
#pragma unroll
      for (int u = 0; u < D / 32; ++u) {
        const int chunk = sub + 16 * u, t = chunk & 3;
        const uint32_t words[4] = {vc[u].x, vc[u].y, vc[u].z, vc[u].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          // D = 128: chunk (h, g, t) = [even w0, even w1, odd w0, odd w1]; D = 64: (g, t) = [h0 even, h0 odd, h1 even, h1 odd]
          const int h = D == 128 ? u >> 1 : x >> 1, o = D == 128 ? x >> 1 : x & 1;
          const int g = D == 128 ? (chunk >> 2) & 7 : chunk >> 2;
          const int d8 = D == 128 ? 2 * g + (x & 1) : g;  // which 8 dims
          const int tok = (tid & ~15) + 8 * h + 2 * t + o;
          *reinterpret_cast<uint4*>(sV + st * KVB + (d8 >> 3) * 16384 + tok * 128 + (((d8 & 7) ^ (tok & 7)) << 4)) =
              values8(words[x], s2[h][o], m2[h][o]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.v_full[st]);
      fetch_v(tile, j + 1);
    }
    kq += (uint32_t)w.steps;
    return true;
  });
}

// ---- one thread: the products, the tiles in turn, so that one's softmax runs while the other multiplies ----
template <int D>
__device__ __forceinline__ void tc_products(const AttendArgs& a, int chunks, TcShared& sh, unsigned char* sQ, unsigned char* sK,
                                            unsigned char* sV, bool* bad) {
  constexpr int QB = TcSmem<D>::Q, KVB = TcSmem<D>::KV;
  constexpr uint32_t bf16_ab = (1u << 7) | (1u << 10);
  constexpr uint32_t id_s = f16_idesc(128, TC_KV) & ~bf16_ab, id_o = (f16_idesc(128, D) & ~bf16_ab) | (1u << 16);
  const uint32_t tmem = sh.tmem;
  const uint64_t dq = sw128_desc(smem_u32(sQ)), dk = sw128_desc(smem_u32(sK));
  const uint64_t dv = sw128_mn_desc(smem_u32(sV), 16384);
  uint32_t q = 0, items = 0;  // steps so far
  auto scores = [&](int i, uint32_t st) {
    const uint64_t x = dq + (uint64_t)(i * (QB >> 4)), k = dk + (uint64_t)(st * (KVB >> 4));
#pragma unroll
    for (int u = 0; u < D / 16; ++u) {
      const uint64_t at = (uint64_t)((u >> 2) * 1024 + (u & 3) * 2);
      tc5_mma(tmem + i * 128, x + at, k + at, id_s, u != 0);
    }
    tc5_commit(&sh.s_full[i]);
  };
  tc_each(a, chunks, sh, bad, [&](const TcWork& w) {
    const int steps = w.steps;
    if (steps == 0) return true;
    if (!mbar_wait(&sh.q_full, items & 1u) || !mbar_wait(&sh.k_full[q & 1u], (q / 2) & 1u)) return false;
    ++items;
    tc5_fence_after();
#pragma unroll 1
    for (int i = 0; i < 2; ++i) scores(i, q & 1u);
#pragma unroll 1
    for (int j = 0; j < steps; ++j, ++q) {
      const uint32_t st = q & 1u, nx = st ^ 1u;
      if (!mbar_wait(&sh.v_full[st], (q / 2) & 1u)) return false;
      const uint64_t v = dv + (uint64_t)(st * (KVB >> 4));
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (!mbar_wait(&sh.p_full[i], q & 1u)) return false;
        tc5_fence_after();
#pragma unroll
        for (int u = 0; u < TC_KV / 16; ++u)
          tc5_mma_ta(tmem + 256 + i * D, tmem + i * 128 + 8 * u, v + (uint64_t)(u * 128), id_o, (j | u) != 0);
        tc5_commit(&sh.o_full[i]);
        if (j + 1 < steps) {
          if (i == 0 && !mbar_wait(&sh.k_full[nx], ((q + 1) / 2) & 1u)) return false;
          // products into different accumulators are not ordered: O has to have taken the P that these scores overwrite
          if (!mbar_wait(&sh.o_full[i], q & 1u)) return false;
          tc5_fence_after();
          scores(i, nx);
        }
      }
    }
    return true;
  });
  // nothing of the tensor core's may be pending when its memory is freed
  tc5_commit(&sh.done);
  mbar_wait(&sh.done, 0);
}

// Registers: 512 threads start with 128 each; 128 (2 x 168 + 96 + 80) = 512 x 128.
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void less_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

template <int D>
__global__ void __launch_bounds__(TC_NT, 1) attend_tc_kernel(AttendArgs a, int chunks) {
  extern __shared__ unsigned char tc_dyn[];
  __shared__ __align__(16) TcShared sh;
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tc_dyn) + 1023) & ~uintptr_t(1023));
  unsigned char* sQ = sm;
  unsigned char* sK = sm + 2 * TcSmem<D>::Q;
  unsigned char* sV = sK + 2 * TcSmem<D>::KV;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(&sh.q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.k_full[i], 4);
      mbar_init(&sh.v_full[i], 4);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_full[i], 1);
    }
    mbar_init(&sh.done, 1);
    sh.fail = 0;
    fence_mbar_init();
  }
  if (warp == 12) tc5_alloc(&sh.tmem, 512);
  tc5_fence_before();
  __syncthreads();
  tc5_fence_after();
  bool bad = false;
  if (warp < 8) {
    more_registers<168>();
    tc_softmax<D>(a, chunks, sh, sQ, &bad);
  } else if (warp < 12) {
    less_registers<96>();
    tc_decode<D>(a, chunks, sh, sK, sV, &bad);
  } else {
    less_registers<80>();
    if (threadIdx.x == 12 * 32) tc_products<D>(a, chunks, sh, sQ, sK, sV, &bad);
  }
  if (bad) atomicOr(a.err, DERR_BOUNDS);
  tc5_fence_before();
  __syncthreads();
  if (sh.fail && threadIdx.x == 0) atomicOr(a.err, DERR_TIMEOUT);
  if (warp == 12) tc5_dealloc(sh.tmem, 512);
}

}  // namespace

void launch_attend_tc(const AttendArgs& a, const AttendShape& s, int chunks, cudaStream_t st) {
  static OncePerDevice once;
  once([] {
    cudaFuncSetAttribute(attend_tc_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<64>::BYTES);
    cudaFuncSetAttribute(attend_tc_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<128>::BYTES);
  });
  const int64_t tiles = ceil_div((int64_t)s.max_q * (s.q_heads / s.kv_heads), TC_ROWS);
  const dim3 grid((unsigned)(std::min<int64_t>(tiles, 1 << 20) * chunks), (unsigned)s.kv_heads,
                  (unsigned)std::min(s.num_seqs, 65535));
  if (s.D == 128) attend_tc_kernel<128><<<grid, TC_NT, TcSmem<128>::BYTES, st>>>(a, chunks);
  else attend_tc_kernel<64><<<grid, TC_NT, TcSmem<64>::BYTES, st>>>(a, chunks);
  count_launch();
}

}  // namespace kl
