// attend_tc.cu -- attention over the paged 4-bit cache for many rows (prompt
// chunks), on tcgen05.  Definitions are in attend.cu.
//
// One block takes 256 rows (token, query head) of one key head as two tiles of
// 128, so that one tile multiplies while the other takes its softmax:
//  * warps 0-3 and 4-7: softmax of tile 0 and 1, one row per thread, straight
//    from tensor memory; P goes back there as bf16, over the scores that it
//    came from; O is rescaled in place only when a row's maximum has risen by
//    more than 2^8;
//  * warps 8-11: the next 128 keys and values, codes read from global memory
//    one tile ahead, turned into bf16 (s c + m in one rounding) and written to
//    shared memory in the tensor core's swizzled layouts, K with D contiguous,
//    V as it stands (its tokens are the product's K, "MN-major");
//  * warp 12: issues S_i = Q_i . K^T and O_i += P_i . V in the order
//    PV_0, S_0, PV_1, S_1 of each step, so the scores' completion also says
//    that O_i may be rescaled.
// Tensor memory: S_0, S_1 (128 columns each), O_0, O_1 (D columns each).
//
// Per 128 keys and 256 rows at D = 128 the tensor cores need 2048 cycles and
// the 32768 exponentials as many of the special function units.
#include "attend.cuh"
#include "engine.h"
#include "tcgen05.cuh"

namespace kl {
namespace {

constexpr int TC_KV = 128;   // keys per step
constexpr int TC_ROWS = 256;  // rows per block
constexpr int TC_NT = 416;   // 13 warps

// MN-major operand, 128-byte swizzle: 64 values of N in 128 bytes, 8 of K in
// 1024; the next 64 of N are lbo bytes on, the next 8 of K 1024.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// A from tensor memory (bf16, two values of K per column)
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

// codes in nibbles 0 and 4 of w as bf16 s c + m, one rounding
__device__ __forceinline__ uint32_t value2(uint32_t w, uint32_t s2, uint32_t m2) {
  const uint32_t v = (w & 0x000f000fu) | 0x43004300u;  // 128 + c, exact
  uint32_t c, r;
  asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(c) : "r"(v), "r"(0x43004300u));
  asm("fma.rn.bf16x2 %0, %1, %2, %3;\n" : "=r"(r) : "r"(c), "r"(s2), "r"(m2));
  return r;
}
// the 8 dims of a word as 16 bytes
__device__ __forceinline__ uint4 values8(uint32_t w, uint32_t s2, uint32_t m2) {
  return make_uint4(value2(w, s2, m2), value2(w >> 4, s2, m2), value2(w >> 8, s2, m2), value2(w >> 12, s2, m2));
}
__device__ __forceinline__ bool nan_low(uint32_t pr) { return (pr & 0x7fff0000u) > 0x7f800000u; }  // the minimum is NaN

template <int D>
struct TcSmem {
  static constexpr int Q = 128 * D * 2;   // one tile
  static constexpr int KV = TC_KV * D * 2;  // one stage of K or V
  static constexpr int BYTES = 2 * Q + 4 * KV + 1024;
};

struct TcBars {
  uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_full[2], o_full[2], done;
};
// every lane's answer, so that a warp gives up as one
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(FULL, mbar_wait(bar, parity));
}

// One pair of row tiles of one sequence.
struct TcWork {
  SeqSpan s;
  int rows, r0, first;  // row r is token first + r / group
  int lo, steps;        // keys [lo, lo + 128 steps) cover what the rows see; lo a multiple of 16
  int hi;               // no row sees hi or later
};
__device__ __forceinline__ TcWork tc_work(const AttendArgs& a, int b, int group, bool* bad) {
  TcWork w;
  w.s = seq_span(a.seq, b, a.cache.page_size, bad);
  w.rows = w.s.q_len * group;
  w.first = w.s.kv_len - w.s.q_len;
  return w;
}
__device__ __forceinline__ void tc_range(TcWork& w, int r0, int group, int window) {
  w.r0 = r0;
  const int pos0 = w.first + r0 / group;
  w.hi = w.first + (min(r0 + TC_ROWS, w.rows) - 1) / group + 1;
  w.lo = (window > 0 ? max(0, pos0 - window + 1) : 0) & ~15;
  w.steps = w.hi > w.lo ? (w.hi - w.lo + TC_KV - 1) / TC_KV : 0;
}

template <int D>
__global__ void __launch_bounds__(TC_NT, 1) attend_tc_kernel(AttendArgs a) {
  extern __shared__ unsigned char tc_dyn[];
  __shared__ TcBars bars;
  __shared__ uint32_t tmem_s;
  __shared__ int fail;
  __shared__ __align__(8) unsigned char no_page[4][8];  // by step & 3: the 16-token tiles whose page does not exist
  constexpr int TB = kv4_tile_bytes(D), CODES = kv4_codes(D);
  constexpr int QB = TcSmem<D>::Q, KVB = TcSmem<D>::KV;
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tc_dyn) + 1023) & ~uintptr_t(1023));
  unsigned char* sQ = sm;
  unsigned char* sK = sm + 2 * QB;
  unsigned char* sV = sK + 2 * KVB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, group = a.q_heads / a.cache.kv_heads;
  if (threadIdx.x == 0) {
    mbar_init(&bars.q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], 4);
      mbar_init(&bars.v_full[i], 4);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_empty[i], 1);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 4);
      mbar_init(&bars.o_full[i], 1);
    }
    mbar_init(&bars.done, 1);
    fail = 0;
    fence_mbar_init();
  }
  if (warp == 12) tc5_alloc(&tmem_s, 512);
  tc5_fence_before();
  __syncthreads();
  tc5_fence_after();
  const uint32_t tmem = tmem_s;
  bool bad = false, lost = false;  // lost: a wait gave up, this role ends
  uint32_t kq = 0, items = 0;      // steps and pairs of tiles done

  for (int b = blockIdx.z; b < a.seq.num_seqs && !lost; b += gridDim.z) {
    TcWork w = tc_work(a, b, group, &bad);
    const int tiles = (w.rows + TC_ROWS - 1) / TC_ROWS;
    // the last rows see most: they go first
    for (int rt = (int)gridDim.x - 1 - (int)blockIdx.x; rt < tiles && !lost; rt += gridDim.x) {
      tc_range(w, rt * TC_ROWS, group, a.window);

      if (warp < 8) {
        // ------------------------------------------------ softmax: one row per thread
        const int i = warp >> 2, r = threadIdx.x & 127, row = w.r0 + i * 128 + r;
        const uint32_t lane_off = (uint32_t)(warp & 3) << 21;
        const uint32_t tS = tmem + i * 128 + lane_off, tO = tmem + 256 + i * D + lane_off;
        const bool live = row < w.rows;
        const int64_t tok = w.s.row + row / group;
        const int head = kvh * group + row % group;
        if (w.steps > 0) {  // the row of Q, K-major with the 128-byte swizzle; a negative scale goes into its sign
          const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
          const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q.p) + tok * a.q.token + head * a.q.head;
          unsigned char* to = sQ + i * QB + r * 128;
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (live) {
              if (a.q.vec) {
                v = reinterpret_cast<const uint4*>(q)[c];
              } else {
                const unsigned short* u = reinterpret_cast<const unsigned short*>(q) + 8 * c;
                v = make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16,
                               u[6] | (uint32_t)u[7] << 16);
              }
              v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
            }
            *reinterpret_cast<uint4*>(to + (c >> 3) * 16384 + (((c & 7) ^ (r & 7)) << 4)) = v;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.q_full);
        }
        const float scl = fabsf(a.scale) * 1.4426950408889634f;
        const int pos = w.first + row / group;
        const int pos_first = w.first + (w.r0 + i * 128) / group;                         // of this tile's rows
        const int pos_last = w.first + (min(w.r0 + i * 128 + 128, max(w.rows, 1)) - 1) / group;
        float ref = 0.f, lift = -INFINITY, l0 = 0.f, l1 = 0.f;
        for (int j = 0; j < w.steps; ++j) {
          if (!warp_wait(&bars.s_full[i], (kq + j) & 1u)) {
            lost = true;
            break;
          }
          tc5_fence_after();
          const int k0 = w.lo + j * TC_KV;
          const int from = a.window > 0 ? pos - a.window + 1 - k0 : 0, to = pos - k0;  // columns [from, to] are seen
          const uint2 none2 = *reinterpret_cast<const uint2*>(no_page[(kq + j) & 3u]);
          const bool holes = (none2.x | none2.y) != 0;
          const bool partial = k0 + TC_KV - 1 > pos_first || (a.window > 0 && k0 <= pos_last - a.window) || holes;
          auto unseen = [&](int col) {
            return col > to || col < from || (holes && no_page[(kq + j) & 3u][col >> 4]);
          };
          float top = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t v[32];
            tc5_ld32(tS + 32 * c, v);
            tc5_ld_wait();
            if (partial) {
#pragma unroll
              for (int u = 0; u < 32; ++u)
                if (unseen(32 * c + u)) v[u] = 0xff800000u;
            }
#pragma unroll
            for (int u = 0; u < 32; ++u) top = fmaxf(top, __uint_as_float(v[u]));
          }
          const float x = top == -INFINITY ? -INFINITY : top * scl;
          if (__any_sync(FULL, x > lift)) {
            const bool none = lift == -INFINITY;
            const float now = x > lift - 8.f || none ? x : ref;
            float keep = 1.f;
            if (now != -INFINITY) {
              keep = none ? 1.f : exp2_fast(ref - now);
              ref = now;
              lift = now + 8.f;
            }
            l0 *= keep;
            l1 *= keep;
            if (j > 0) {
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t v[32];
                tc5_ld32(tO + 32 * c, v);
                tc5_ld_wait();
#pragma unroll
                for (int u = 0; u < 32; ++u) v[u] = __float_as_uint(__uint_as_float(v[u]) * keep);
                tc5_st16(tO + 32 * c, v);
                tc5_st16(tO + 32 * c + 16, v + 16);
              }
            }
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t v[32], pk[16];
            tc5_ld32(tS + 32 * c, v);
            tc5_ld_wait();
            if (partial) {
#pragma unroll
              for (int u = 0; u < 32; ++u)
                if (unseen(32 * c + u)) v[u] = 0xff800000u;
            }
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const float y0 = exp2_fast(fmaf(__uint_as_float(v[2 * u]), scl, -ref));
              const float y1 = exp2_fast(fmaf(__uint_as_float(v[2 * u + 1]), scl, -ref));
              l0 += y0;
              l1 += y1;
              pk[u] = pack_bf16(y0, y1);
            }
            tc5_st16(tS + 16 * c, pk);
          }
          tc5_st_wait();
          tc5_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.p_full[i]);
        }
        if (!lost && w.steps > 0) {
          if (warp_wait(&bars.o_full[i], items & 1u)) tc5_fence_after();
          else lost = true;
        }
        if (!lost) {
          const float l = l0 + l1, inv = l == 0.f ? 0.f : 1.f / l;
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out.p) + tok * a.out.token + head * a.out.head;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t v[32];
            if (w.steps > 0) {
              tc5_ld32(tO + 32 * c, v);
              tc5_ld_wait();
            } else {
#pragma unroll
              for (int u = 0; u < 32; ++u) v[u] = 0u;
            }
            if (live) {
              float y[32];
#pragma unroll
              for (int u = 0; u < 32; ++u) y[u] = l == 0.f ? 0.f : __uint_as_float(v[u]) * inv;
#pragma unroll
              for (int u = 0; u < 4; ++u) store8_bf16(out + 32 * c + 8 * u, a.out.vec, y + 8 * u);
            }
          }
          tc5_fence_before();  // the next rows' first product overwrites O
        }
      } else if (warp < 12) {
        // ------------------------------------------------ keys and values
        const int tid = threadIdx.x - 256, sub = tid & 15;
        const int32_t* table = a.seq.table + b * a.seq.table_ld;
        const int ps = a.cache.page_size, tpp = a.cache.tiles_per_page;
        uint4 kc[4], vc[4], vp[2];
        uint2 kp;
        bool hole = false;
        auto page_of = [&](int j) {
          const int n = w.lo + j * TC_KV + (tid & ~15);
          return j < w.steps && n < w.hi ? table[n / ps] : -1;
        };
        auto fetch = [&](int j, int32_t page) {
          const int n = w.lo + j * TC_KV + (tid & ~15);
          if (j < w.steps && n < w.hi && (page < 0 || page >= a.cache.num_pages)) {
            bad = true;
            page = -1;
          }
          if (page < 0) {
#pragma unroll
            for (int u = 0; u < 4; ++u) kc[u] = vc[u] = make_uint4(0, 0, 0, 0);
            vp[0] = vp[1] = make_uint4(0, 0, 0, 0);
            kp = make_uint2(0, 0);
            hole = j < w.steps && n < w.hi;
            return;
          }
          hole = false;
          const unsigned char* tile = kv4_tile(a.cache, TB, page, kvh, (n >> 4) % tpp);
          const unsigned char* codes = tile + CODES;
          const unsigned char* pr = tile + 2 * CODES;
          if (D == 128) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              kc[u] = *reinterpret_cast<const uint4*>(tile + sub * 64 + u * 16);
              vc[u] = *reinterpret_cast<const uint4*>(codes + (sub + 16 * u) * 16);
            }
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const uint2 x = *reinterpret_cast<const uint2*>(tile + (sub & 7) * 64 + u * 16 + (sub >> 3) * 8);
              kc[u] = make_uint4(x.x, x.y, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) vc[u] = *reinterpret_cast<const uint4*>(codes + (sub + 16 * u) * 16);
          }
          kp = *reinterpret_cast<const uint2*>(pr + sub * 8);
#pragma unroll
          for (int h = 0; h < 2; ++h) vp[h] = *reinterpret_cast<const uint4*>(pr + (8 * h + 2 * (sub & 3)) * 8);
        };
        int32_t next = page_of(1);
        fetch(0, page_of(0));
        for (int j = 0; j < w.steps; ++j) {
          const uint32_t q = kq + j, st = q & 1u;
          // ---- K: this thread's token, D contiguous ----
          if (q >= 2 && !warp_wait(&bars.k_empty[st], (q / 2 - 1) & 1u)) {
            lost = true;
            break;
          }
          // four slots: a step's is written again when the step three on has its scores, after this one's softmax
          if (sub == 0) no_page[q & 3u][tid >> 4] = hole;
          {
            // a value that is not finite: the key becomes NaN for whoever sees it, the value zero, since a
            // product with it reaches rows that do not
            const bool nan = nan_low(kp.x) || nan_low(kp.y);
            const uint32_t s = nan ? 0u : kp.x & 0xffffu, m = nan ? 0x7fffu : kp.x >> 16;
            const uint32_t s2 = s | s << 16, m2 = m | m << 16;
            unsigned char* to = sK + st * KVB + tid * 128;
#pragma unroll
            for (int u = 0; u < D / 8; ++u) {
              const uint32_t word = D == 128 ? (&kc[u >> 2].x)[u & 3] : (&kc[u >> 1].x)[u & 1];
              *reinterpret_cast<uint4*>(to + (u >> 3) * 16384 + (((u & 7) ^ (tid & 7)) << 4)) = values8(word, s2, m2);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.k_full[st]);
          // ---- V: 16-byte chunks of the codes; two tokens each ----
          if (q >= 2 && !warp_wait(&bars.v_empty[st], (q / 2 - 1) & 1u)) {
            lost = true;
            break;
          }
#pragma unroll
          for (int u = 0; u < D / 32; ++u) {
            const int chunk = sub + 16 * u, t = chunk & 3;
            const uint32_t words[4] = {vc[u].x, vc[u].y, vc[u].z, vc[u].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              // D = 128: chunk (h, g, t) = [even w0, even w1, odd w0, odd w1]; D = 64: (g, t) = [h0 e, h0 o, h1 e, h1 o]
              const int h = D == 128 ? u >> 1 : x >> 1, o = D == 128 ? x >> 1 : x & 1;
              const int g = D == 128 ? (chunk >> 2) & 7 : chunk >> 2;
              const int d8 = D == 128 ? 2 * g + (x & 1) : g;  // which 8 dims
              const uint32_t k2 = o ? vp[h].z : vp[h].x, v2 = o ? vp[h].w : vp[h].y;
              const bool nan = nan_low(k2) || nan_low(v2);
              const uint32_t s = nan ? 0u : v2 & 0xffffu, m = nan ? 0u : v2 >> 16;
              const int tok = (tid & ~15) + 8 * h + 2 * t + o;
              *reinterpret_cast<uint4*>(sV + st * KVB + (d8 >> 3) * 16384 + tok * 128 + (((d8 & 7) ^ (tok & 7)) << 4)) =
                  values8(words[x], s | s << 16, m | m << 16);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.v_full[st]);
          fetch(j + 1, next);
          next = page_of(j + 2);
        }
      } else if (lane == 0 && w.steps > 0) {
        // ------------------------------------------------ the products
        const uint32_t id_s = f16_idesc(128, TC_KV), id_o = f16_idesc(128, D) | (1u << 16);
        auto scores = [&](int i, uint32_t st) {
          const uint64_t dq = sw128_desc(smem_u32(sQ + i * QB)), dk = sw128_desc(smem_u32(sK + st * KVB));
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t off = (uint64_t)((k >> 2) * 1024 + (k & 3) * 2);
            tc5_mma(tmem + i * 128, dq + off, dk + off, id_s, k != 0);
          }
          tc5_commit(&bars.s_full[i]);
        };
        lost = !mbar_wait(&bars.q_full, items & 1u) || !mbar_wait(&bars.k_full[kq & 1u], (kq / 2) & 1u);
        if (!lost) {
          tc5_fence_after();
          scores(0, kq & 1u);
          scores(1, kq & 1u);
          tc5_commit(&bars.k_empty[kq & 1u]);
        }
        for (int j = 0; j < w.steps && !lost; ++j) {
          const uint32_t q = kq + j, st = q & 1u, nx = st ^ 1u;
          if (!mbar_wait(&bars.v_full[st], (q / 2) & 1u)) {
            lost = true;
            break;
          }
          for (int i = 0; i < 2; ++i) {
            if (!mbar_wait(&bars.p_full[i], q & 1u)) {
              lost = true;
              break;
            }
            tc5_fence_after();
            const uint64_t dv = sw128_mn_desc(smem_u32(sV + st * KVB), 16384);
#pragma unroll
            for (int k = 0; k < TC_KV / 16; ++k)
              tc5_mma_ta(tmem + 256 + i * D, tmem + i * 128 + 8 * k, dv + (uint64_t)(k * 128), id_o, (j | k) != 0);
            if (i == 1) tc5_commit(&bars.v_empty[st]);
            if (j + 1 < w.steps) {
              if (i == 0 && !mbar_wait(&bars.k_full[nx], ((q + 1) / 2) & 1u)) {
                lost = true;
                break;
              }
              tc5_fence_after();
              scores(i, nx);
              if (i == 1) tc5_commit(&bars.k_empty[nx]);
            } else {
              tc5_commit(&bars.o_full[i]);
            }
          }
        }
      }
      if (lost) atomicExch(&fail, 1);
      kq += (uint32_t)w.steps;
      if (w.steps > 0) ++items;
    }
  }
  if (warp == 12 && lane == 0) {  // nothing of the tensor core's may be pending when its memory is freed
    tc5_commit(&bars.done);
    mbar_wait(&bars.done, 0);
  }
  tc5_fence_before();
  __syncthreads();
  if (fail && threadIdx.x == 0) atomicOr(a.err, DERR_TIMEOUT);
  if (bad) atomicOr(a.err, DERR_BOUNDS);
  if (warp == 12) tc5_dealloc(tmem, 512);
}

}  // namespace

void launch_attend_tc(const AttendArgs& a, const AttendShape& s, cudaStream_t st) {
  static OncePerDevice once;
  once([] {
    cudaFuncSetAttribute(attend_tc_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<64>::BYTES);
    cudaFuncSetAttribute(attend_tc_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<128>::BYTES);
  });
  const int64_t tiles = ceil_div((int64_t)s.max_q * (s.q_heads / s.kv_heads), TC_ROWS);
  const dim3 grid((unsigned)std::min<int64_t>(tiles, 1 << 20), (unsigned)s.kv_heads,
                  (unsigned)std::min(s.num_seqs, 65535));
  if (s.D == 128) attend_tc_kernel<128><<<grid, TC_NT, TcSmem<128>::BYTES, st>>>(a);
  else attend_tc_kernel<64><<<grid, TC_NT, TcSmem<64>::BYTES, st>>>(a);
  count_launch();
}

}  // namespace kl
