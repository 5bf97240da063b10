// attend.cu -- attention of a call's new tokens over the paged 4-bit cache
// (kv4.cuh): o = softmax(scale * q . K^T) . V over the keys that a token sees,
// K = ks c + km, V = vs c + vm.  Token i of a sequence (0-based over its whole
// length) sees tokens j <= i, and with a window w only i - w < j.  A token
// that sees nothing gets zeros.
//
// The steps stay out of the codes: with one step and minimum per head vector,
//   q . K_j = ks_j (q . c_j) + km_j sum(q),
//   sum_j p_j V_j = sum_j (p_j vs_j) c_j + sum_j p_j vm_j,
// so the tensor cores multiply bare codes 0..15, and steps and minima touch
// one score and one probability per key, not D values.
#include "attend.cuh"
#include "engine.h"
#include "pdl.cuh"
#include "tcgen05.cuh"

namespace kl {
namespace {

constexpr int AT_W = 4;       // warps per block
constexpr int AT_STAGES = 3;  // pairs of tiles of a warp's ring

struct SplitPlan {
  int least;      // fewest tokens per block, a multiple of 16 AT_W
  int chunks;     // blocks along a sequence
  int row_tiles;  // blocks along a sequence's rows
};
// Shared memory of a block: the rings, and where the warps join.
template <int D, int NR>
constexpr int split_smem() {
  constexpr int ring = AT_W * AT_STAGES * 2 * kv4_tile_bytes(D), join = AT_W * 8 * NR * D * 4;
  return ring > join ? ring : join;
}

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the 8 x 8 matrix of 16-bit values whose row g, columns 2t, 2t + 1 lane (g, t) holds, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Few rows: decode steps and drafts.  One block takes a chunk of a sequence for
// up to 8 NR rows (token, query head of one key head); its warps take the
// chunk's 16-token tiles in turn, each through a ring of its own filled by
// bulk copies, and join at the end; chunks of a sequence are joined by
// attend_join_kernel.
//
// S^T = K . Q^T and O^T = V^T . P^T, so keys fill the 16 rows of a matrix
// fragment and query rows its 8 columns.  A code is used as it stands: its
// nibble in an f16 register is the number c 2^-24, the second nibble of a byte
// 16 c 2^-24 (q, or that dim of O, divided by 16), exact in the product, so a
// word of 8 codes costs five logic instructions.  q is scaled by a power of two
// into f16's range, which loses what is below 2^-37 of the row's largest;
// probabilities go in times their value's step and a power of two 2^-E that
// keeps the largest so far within f16, rounded to 11 bits (2^-11 at most), and
// what is 2^-33 of the largest or less to none.  That is bits fewer than the
// inputs have, and shows beside the output's own bf16: against 64 bits 0.0018 of
// the output's size (0.0019 over 131071 tokens) where bf16 alone gives 0.0017.
// References are whole numbers: where one rises, E falls as much and O stays as
// it is, so that large values whose keys have been outdone leave the range to
// what counts.  Sums, maxima and O are f32.
//
// D + 8 bytes a token and key head.  64 sequences of up to 16384 tokens, D = 128,
// 8 key heads of 4 rows: 146 us, 4.0 TB/s of 6.4; one of 131071: 43 us, 3.3 TB/s.
// Nothing is saturated: of 4 issue slots 2.3 are taken, logic (of the nibbles,
// about half of 300 instructions a warp for 16 tokens) 57% of its rate, memory
// 44%.  With 16 warps a processor, which 127 registers allow, the chains from a
// score to its weight's product are waited for.
template <int D, int NR>
__global__ void __launch_bounds__(AT_W * 32, NR == 1 ? 4 : 3) attend_split_kernel(AttendArgs a, SplitPlan p) {
  constexpr int TB = kv4_tile_bytes(D), CODES = kv4_codes(D);
  constexpr int KW = D / 32;  // words of K per lane and token
  constexpr int MT = D / 16;  // O^T fragments
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ uint64_t full[AT_W][AT_STAGES];
  __shared__ int tile_ok[AT_W][AT_STAGES][2];
  __shared__ float2 ml[AT_W][8 * NR];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, group = a.q_heads / a.cache.kv_heads, ps = a.cache.page_size;
  const int chunk_id = blockIdx.x / p.row_tiles;
  unsigned char* mine = ring + warp * AT_STAGES * 2 * TB;
  if (lane < AT_STAGES) mbar_init(&full[warp][lane], 2);
  fence_mbar_init();
  __syncthreads();
  // without begin_next(): blocks of the join that wait beside these cost more than their launch (8.9 against 7.5 us)
  after_before();
  uint32_t used = 0;  // pairs of tiles that this warp has put through its ring
  const float log2e = 1.4426950408889634f;
  // The longest sequence's tokens are shared out evenly, the others' cut alike.  Its length is looked up, since hints
  // are the cache's whole capacity in a captured loop.  With exact hints and with such of 131072, us: one token of 777
  // 7.9 and 9.9 (chunks by the hint alone 7.6 and 15.2), of 8000 11.0 and 13.5 (10.6 and 22.5), 64 sequences of 8000
  // 126 and 126 (124 and 152), 8 of up to 30000 30 and 30 (30 and 137).
  uint32_t share = p.chunks > 1 ? 0u : p.least;
  const int some = p.chunks > 1 && lane < a.seq.num_seqs ? a.seq.kv_len[lane] : 0;

  for (int b = blockIdx.z; b < a.seq.num_seqs; b += gridDim.z) {
    bool bad = false;
    const SeqSpan s = seq_span(a.seq, b, ps, &bad);
    if (bad && threadIdx.x == 0) atomicOr(a.err, DERR_BOUNDS);
    if (share == 0) {
      int most = some;
      for (int i = lane + 32; i < a.seq.num_seqs; i += 32) most = max(most, a.seq.kv_len[i]);
      uint32_t longest = (uint32_t)max(0, __reduce_max_sync(FULL, most));
      if (a.window > 0) longest = min(longest, (uint32_t)a.window + 8 * NR + 17);
      share = max((uint32_t)p.least, ((longest + p.chunks - 1) / p.chunks + 16 * AT_W - 1) & ~(16 * AT_W - 1));
    }
    const int rows = s.q_len * group, first = s.first;  // row r is token first + r / group
    for (int r0 = (blockIdx.x % p.row_tiles) * 8 * NR; r0 < rows; r0 += p.row_tiles * 8 * NR) {
      // tokens that some row of this tile sees: [lo, hi), this block's share [k0, k1)
      const int pos0 = first + r0 / group, pos1 = first + (min(r0 + 8 * NR, rows) - 1) / group, hi = min(pos1 + 1, s.kv_len);
      const int lo = window_from(a.window, pos0) & ~15;
      const int span = max(0, hi - lo);
      // what does not fit is the last chunk's
      const int64_t at0 = lo + (int64_t)chunk_id * share, at1 = chunk_id + 1 < p.chunks ? at0 + share : hi;
      const int k0 = (int)min((int64_t)hi, at0), k1 = (int)max((int64_t)k0, min((int64_t)hi, at1));
      const int t0 = k0 >> 4, tiles = (k1 - k0 + 15) >> 4;  // k0 is a multiple of 16 wherever tiles > 0
      if (tiles == 0 && p.chunks > 1) {  // a chunk behind the sequence's end, as hints make them
        for (int r = r0 + threadIdx.x; r < min(r0 + 8 * NR, rows); r += AT_W * 32)
          reinterpret_cast<float2*>(a.scratch)[((int64_t)chunk_id * a.seq.num_tokens + s.row + r / group) * a.q_heads + kvh * group +
                                               r % group] = make_float2(-INFINITY, 0.f);
        continue;
      }
      // this warp's tiles are warp, warp + AT_W, ..; it takes them in pairs, for two chains of everything
      const int mine_n = tiles > warp ? (tiles - warp + AT_W - 1) / AT_W : 0, n = (mine_n + 1) / 2;

      // ---- the ring's first fills: lane i takes the warp's tile i ----
      const int32_t* table = a.seq.table + b * a.seq.table_ld;
      const int tpp = a.cache.tiles_per_page;
      const int64_t page_bytes = (int64_t)a.cache.kv_heads * tpp * TB;
      const unsigned char* heads = a.cache.base + (int64_t)kvh * tpp * TB;
      auto issue = [&](int i, int col, int32_t page) {  // by a lane, for tile i; beyond the last: nothing to see
        const uint32_t st = (used + (i >> 1)) % AT_STAGES;
        const int off = t0 + warp + i * AT_W - col * tpp;
        const bool ok = i < mine_n && page >= 0 && page < a.cache.num_pages;
        tile_ok[warp][st][i & 1] = ok;
        if (ok) {
          mbar_arrive_expect_tx(&full[warp][st], TB);
          bulk_load(mine + (2 * st + (i & 1)) * TB, heads + page * page_bytes + off * TB, TB, &full[warp][st]);
        } else {
          if (i < mine_n) atomicOr(a.err, DERR_BOUNDS);
          mbar_arrive(&full[warp][st]);
        }
      };
      if (lane < 2 * AT_STAGES && lane < 2 * n) {
        const int col = lane < mine_n ? kv4_column(a.cache, t0 + warp + lane * AT_W) : 0;
        issue(lane, col, lane < mine_n ? table[col] : 0);
      }

      // ---- q: row g's dims [t D/4, (t+1) D/4), scaled by a power of two ----
      uint32_t qf[NR][2 * KW][2];
      float f[NR][2], qs[NR][2];  // of rows 2t, 2t + 1: what a product of codes is worth, and sum(q), in units of log2
      int pos[NR][2];
      bool big = false;  // a row above 2^113: 2^12 of what its products are worth goes to the keys' steps and minima
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const int row = r0 + 8 * r + g;
        float x[D / 4], top = 0.f, sum = 0.f;
        bool fin = true;
        if (row < rows) {
          const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(a.q.p) + (s.row + row / group) * a.q.token +
                                    (kvh * group + row % group) * a.q.head + t * (D / 4);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) load8_bf16(qp + 8 * i, a.q.vec, x + 8 * i);
        } else {
#pragma unroll
          for (int i = 0; i < D / 4; ++i) x[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
          top = fmaxf(top, fabsf(x[i]));
          fin = fin && finite_f(x[i]);
        }
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
        const int e = max(-114, min(126, 13 - ((int)(__float_as_uint(top) >> 23) - 127)));
        const float up = __uint_as_float((uint32_t)(e + 127) << 23), up16 = up * 0.0625f;
        big = big || e < -100;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) sum = fmaf(x[i], up, sum);
        sum += __shfl_xor_sync(FULL, sum, 1);
        sum += __shfl_xor_sync(FULL, sum, 2);
        const unsigned bads = __ballot_sync(FULL, !fin);
        fin = ((bads >> (4 * g)) & 15u) == 0;
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float* y = x + 8 * w + 4 * h;
            qf[r][2 * w + h][0] = fin ? pack_f16(y[0] * up, y[1] * up) : 0u;
            qf[r][2 * w + h][1] = fin ? pack_f16(y[2] * up16, y[3] * up16) : 0u;
          }
        const float worth = __uint_as_float((uint32_t)(12 - e + 127) << 23) * (a.scale * log2e);
        const float total = fin ? sum * (a.scale * log2e) * __uint_as_float((uint32_t)(127 - e) << 23) * 0x1p-12f
                                : __int_as_float(0x7fffffff);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f[r][i] = __shfl_sync(FULL, worth, 4 * (2 * t + i));
          qs[r][i] = __shfl_sync(FULL, total, 4 * (2 * t + i));
          pos[r][i] = first + (r0 + 8 * r + 2 * t + i) / group;
        }
      }
      big = __any_sync(FULL, big);
      const float key_up = big ? 0x1p12f : 1.f;
      if (!big) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int i = 0; i < 2; ++i) f[r][i] *= 0x1p12f, qs[r][i] *= 0x1p12f;
      }
      const int see_all_to = pos0;  // every row of the tile sees tokens up to here ..
      const int see_all_from = window_from(a.window, pos1);  // .. from here

      float o[MT][NR][4], l[NR][2], vb[NR][2], ref[NR][2], lift[NR][2];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[m][r][i] = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[r][i] = vb[r][i] = ref[r][i] = 0.f;
          lift[r][i] = -INFINITY;  // a score above this moves the row's reference
        }
      }
      float down[NR][2];  // 2^-E of a row's weights; first so large that any that matters asks for another
#pragma unroll
      for (int r = 0; r < NR; ++r) down[r][0] = down[r][1] = 8.507059e37f;  // 2^126
      // the refills' lanes, one for each of two tiles, have the next one's page at hand
      int next = 2 * AT_STAGES + lane, next_col = 0;
      int32_t next_page = 0;
      if (lane < 2 && next < mine_n) {
        next_col = kv4_column(a.cache, t0 + warp + next * AT_W);
        next_page = table[next_col];
      }

      for (int i = 0; i < n; ++i) {
        const uint32_t st = (used + i) % AT_STAGES;
        if (!mbar_wait(&full[warp][st], ((used + i) / AT_STAGES) & 1u)) {
          atomicOr(a.err, DERR_TIMEOUT);
          // no copy may land where the warps are about to join
          for (int k = i; k < min(n, i + AT_STAGES); ++k)
            mbar_wait(&full[warp][(used + k) % AT_STAGES], ((used + k) / AT_STAGES) & 1u);
          break;
        }
        const unsigned char* tile = mine + 2 * st * TB;
        uint32_t ve[2][2][KW / 2], vo[2][2][KW / 2];
        float x[2][NR][4], vs[2][2], vm[2][2];  // x[.][r][2 k + u]: key g + 8 k of the tile, row 2t + u
        bool ok[2];
#pragma unroll
        for (int c = 0; c < 2; ++c, tile += TB) {
          uint32_t kw[2][KW];
          if (D == 128) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint4 k = *reinterpret_cast<const uint4*>(tile + h * 512 + lane * 16);
              const uint4 v = *reinterpret_cast<const uint4*>(tile + CODES + h * 512 + lane * 16);
              kw[h][0] = k.x; kw[h][1] = k.y; kw[h][KW - 2] = k.z; kw[h][KW - 1] = k.w;
              ve[c][h][0] = v.x; ve[c][h][KW / 2 - 1] = v.y; vo[c][h][0] = v.z; vo[c][h][KW / 2 - 1] = v.w;
            }
          } else {
            const uint4 k = *reinterpret_cast<const uint4*>(tile + lane * 16);
            const uint4 v = *reinterpret_cast<const uint4*>(tile + CODES + lane * 16);
            kw[0][0] = k.x; kw[0][1] = k.y; kw[1][0] = k.z; kw[1][1] = k.w;
            ve[c][0][0] = v.x; vo[c][0][0] = v.y; ve[c][1][0] = v.z; vo[c][1][0] = v.w;
          }
          ok[c] = tile_ok[warp][st][c];
          uint2 pr[2] = {*reinterpret_cast<const uint2*>(tile + 2 * CODES + g * 8),
                         *reinterpret_cast<const uint2*>(tile + 2 * CODES + (g + 8) * 8)};
          if (!ok[c]) pr[0] = pr[1] = make_uint2(0, 0);
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int u = 0; u < 4; ++u) x[c][r][u] = 0.f;
#pragma unroll
          for (int w = 0; w < KW; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t u0 = kw[0][w] >> (8 * h), u1 = kw[1][w] >> (8 * h);
#pragma unroll
              for (int r = 0; r < NR; ++r)
                mma_f16(x[c][r], u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u,
                        qf[r][2 * w + h][0], qf[r][2 * w + h][1]);
            }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float ks = __uint_as_float(pr[k].x << 16) * key_up;
            float km = __uint_as_float(pr[k].x & 0xffff0000u) * key_up;
            vs[c][k] = __uint_as_float(pr[k].y << 16);
            vm[c][k] = __uint_as_float(pr[k].y & 0xffff0000u);
            // a value that is NaN makes the score NaN for whoever sees it, and is nothing to the others
            if (vm[c][k] != vm[c][k]) {
              km = vm[c][k];
              vm[c][k] = 0.f;
            }
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
              for (int u = 0; u < 2; ++u)
                x[c][r][2 * k + u] = fmaf(x[c][r][2 * k + u] * ks, f[r][u], km * qs[r][u]);
          }
        }
        __syncwarp();  // the stage has been read: it is filled again
        if (lane < 2 && i + AT_STAGES < n) {
          issue(next, next_col, next_page);
          next += 2;
          if (next < mine_n) {
            next_col = kv4_column(a.cache, t0 + warp + next * AT_W);
            next_page = table[next_col];
          }
        }

        const int j0 = (t0 + warp + 2 * i * AT_W) * 16;  // the first tile's first key; the second's is 16 AT_W on
        if (j0 + 16 * AT_W + 15 > see_all_to || j0 < see_all_from || !ok[0] || !ok[1]) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int j = j0 + c * 16 * AT_W + g + 8 * (u >> 1), q = pos[r][u & 1];
                if (!ok[c] || j > q || (a.window > 0 && q - j >= a.window)) x[c][r][u] = -INFINITY;
              }
        }
        float top[NR][2];
        bool up = false;
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            top[r][u] = fmaxf(fmaxf(x[0][r][u], x[0][r][2 + u]), fmaxf(x[1][r][u], x[1][r][2 + u]));
            up = up || top[r][u] > lift[r][u];
          }
        if (__any_sync(FULL, up)) {
          // move the references to the maxima seen so far (a probability is at most 2^8 until the next move)
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top[r][u] = fmaxf(top[r][u], __shfl_xor_sync(FULL, top[r][u], d));
              const bool none = lift[r][u] == -INFINITY;
              top[r][u] = ceilf(top[r][u]);
              if ((top[r][u] > ref[r][u] || none) && top[r][u] != -INFINITY) {
                // sums taken with no finite score so far are NaN or zero: both stay what they are
                const float rise = none ? 0.f : fminf(top[r][u] - ref[r][u], 253.f), keep = exp2f(-rise);
                l[r][u] *= keep;
                vb[r][u] *= keep;
                const int room = 253 - (int)(__float_as_uint(down[r][u]) >> 23);  // to 2^126
                if ((int)rise > room) {  // O with what is left of it
                  const float less = exp2f((float)room - rise);
#pragma unroll
                  for (int m = 0; m < MT; ++m) {
                    o[m][r][u] *= less;
                    o[m][r][2 + u] *= less;
                  }
                }
                down[r][u] = __uint_as_float(__float_as_uint(down[r][u]) + ((uint32_t)min((int)rise, room) << 23));
                ref[r][u] = top[r][u];
                lift[r][u] = top[r][u] + 8.f;
              }
            }
        }
        bool heavy = false;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const float y = exp2_fast(x[c][r][u] - ref[r][u & 1]);
              l[r][u & 1] += y;
              vb[r][u & 1] = fmaf(y, vm[c][u >> 1], vb[r][u & 1]);
              x[c][r][u] = y * vs[c][u >> 1];  // the weight of a code
              heavy = heavy || x[c][r][u] * down[r][u & 1] > 32768.f;
            }
        if (__any_sync(FULL, heavy)) {
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float most = fmaxf(fmaxf(x[0][r][u], x[0][r][2 + u]), fmaxf(x[1][r][u], x[1][r][2 + u]));
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(FULL, most, d));
              if (most * down[r][u] > 32768.f) {  // E: this weight at 2^8; later ones may pass it by 2^7
                const int e = max(-126, 8 - ((int)(__float_as_uint(most) >> 23) - 127));
                const float now = __uint_as_float((uint32_t)(e + 127) << 23), keep = now / down[r][u];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                  o[m][r][u] *= keep;
                  o[m][r][2 + u] *= keep;
                }
                down[r][u] = now;
              }
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pb[NR][2];
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              pb[r][k] = transpose8(pack_f16(x[c][r][2 * k] * down[r][0], x[c][r][2 * k + 1] * down[r][1]));
#pragma unroll
          for (int w = 0; w < KW / 2; ++w) {
            uint32_t lo2[2], hi2[2];  // dims 0 2 4 6 and 1 3 5 7 of the word, tokens 2t and 2t + 1 side by side
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              lo2[h] = __byte_perm(ve[c][h][w], vo[c][h][w], 0x5410);
              hi2[h] = __byte_perm(ve[c][h][w], vo[c][h][w], 0x7632);
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const uint32_t mask = d & 1 ? 0x00f000f0u : 0x000f000fu;
              const int s = d & 2 ? 8 : 0;
#pragma unroll
              for (int r = 0; r < NR; ++r)
                mma_f16(o[4 * w + d][r], lo2[0] >> s & mask, hi2[0] >> s & mask, lo2[1] >> s & mask, hi2[1] >> s & mask,
                        pb[r][0], pb[r][1]);
            }
          }
        }
      }
      used += n;

      // ---- join the warps: every warp's rows [8 NR][D] and (reference, sum) in shared memory ----
      __syncthreads();
      float* part = reinterpret_cast<float*>(ring);
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            l[r][u] += __shfl_xor_sync(FULL, l[r][u], d);
            vb[r][u] += __shfl_xor_sync(FULL, vb[r][u], d);
          }
          const int row = 8 * r + 2 * t + u;
          float* at = part + (warp * 8 * NR + row) * D + g * (D / 8);
          const float up = 1.f / down[r][u];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const float f = m & 1 ? 1048576.f : 16777216.f;  // a code is worth 2^-24, or 2^-20
            *reinterpret_cast<float2*>(at + 2 * m) =
                make_float2(fmaf(o[m][r][u] * f, up, vb[r][u]), fmaf(o[m][r][2 + u] * f, up, vb[r][u]));
          }
          if (g == 0) ml[warp][row] = make_float2(lift[r][u] == -INFINITY ? -INFINITY : ref[r][u], l[r][u]);
        }
      __syncthreads();
      for (int e = threadIdx.x; e < 8 * NR * (D / 4); e += AT_W * 32) {
        const int row = e / (D / 4), d = e % (D / 4) * 4;
        if (r0 + row >= rows) continue;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < AT_W; ++w) top = fmaxf(top, ml[w][row].x);
        const float rf = top == -INFINITY ? 0.f : top;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < AT_W; ++w) {
          const float2 v = ml[w][row];
          const float keep = exp2f(v.x - rf);
          const float4 y = *reinterpret_cast<const float4*>(part + (w * 8 * NR + row) * D + d);
          sum = fmaf(keep, v.y, sum);
          acc[0] = fmaf(keep, y.x, acc[0]);
          acc[1] = fmaf(keep, y.y, acc[1]);
          acc[2] = fmaf(keep, y.z, acc[2]);
          acc[3] = fmaf(keep, y.w, acc[3]);
        }
        const int64_t tok = s.row + (r0 + row) / group;
        const int head = kvh * group + (r0 + row) % group;
        if (p.chunks == 1) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          attend_store4(a.out, tok, head, d, acc, inv);
        } else {
          const int64_t at = ((int64_t)chunk_id * a.seq.num_tokens + tok) * a.q_heads + head;
          if (sum != 0.f)
            *reinterpret_cast<float4*>(join_rows(a, p.chunks) + at * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
          if (d == 0) reinterpret_cast<float2*>(a.scratch)[at] = make_float2(top, sum);
        }
      }
      fence_proxy_async_smem();  // the ring, written here by threads, is next written by copies
      __syncthreads();
    }
  }
}

// W warps per (token, query head): the chunks' rows, brought to one reference
// and summed, each warp every W-th chunk, the warps in order.  One warp reads
// 74 chunks in 19 us, a load's latency each; eight, four loads at a time, in 4.
template <int D, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) attend_join_kernel(AttendArgs a, int chunks) {
  constexpr int E = D / 32;
  __shared__ float part[W][D];
  __shared__ float sums[W];
  begin_next();
  after_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, me = W == 1 ? 0 : warp;
  const int64_t i = W == 1 ? (int64_t)blockIdx.x * 4 + warp : (int64_t)blockIdx.x;
  if (i >= (int64_t)a.seq.num_tokens * a.q_heads) return;
  const int64_t tok = i / a.q_heads;
  const int head = (int)(i % a.q_heads);
  if (tok < a.seq.cu_q[0] || tok >= a.seq.cu_q[a.seq.num_seqs]) return;  // a row of no sequence
  const int64_t step = (int64_t)a.seq.num_tokens * a.q_heads;
  const float2* ml = reinterpret_cast<const float2*>(a.scratch) + i;
  const float* rows = join_rows(a, chunks) + i * D + lane * E;
  float top = -INFINITY;
  for (int c = lane; c < chunks; c += 32) top = fmaxf(top, ml[c * step].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, d));
  const float rf = top == -INFINITY ? 0.f : top;
  float sum = 0.f, acc[E] = {};
  for (int c0 = me; c0 < chunks; c0 += 4 * W) {
    float2 v[4];
    float r[4][E];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + u * W;
      v[u] = c < chunks ? ml[c * step] : make_float2(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        // a chunk that saw nothing wrote no row
        const float2 x = v[u].y != 0.f ? *reinterpret_cast<const float2*>(rows + c * step * D + e) : make_float2(0.f, 0.f);
        r[u][e] = x.x;
        r[u][e + 1] = x.y;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float keep = v[u].y != 0.f ? exp2f(v[u].x - rf) : 0.f;
      sum = fmaf(keep, v[u].y, sum);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(keep, r[u][e], acc[e]);
    }
  }
  if (W > 1) {
    if (lane == 0) sums[me] = sum;
#pragma unroll
    for (int e = 0; e < E; ++e) part[me][lane * E + e] = acc[e];
    __syncthreads();
    if (warp > 0) return;
    sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      sum += sums[w];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += part[w][lane * E + e];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out.p) + tok * a.out.token + head * a.out.head + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = __float2bfloat16_rn(acc[e] * inv);
}

// The longest stretch of keys that a tile of rows may see.
int64_t plan_span(const AttendShape& s, int rows_per_tile) {
  if (s.window <= 0) return s.max_kv;
  return std::min<int64_t>(s.max_kv, (int64_t)s.window + ceil_div(rows_per_tile, s.q_heads / s.kv_heads) + 16);
}

SplitPlan split_plan(const AttendShape& s) {
  const int64_t rows = (int64_t)s.max_q * (s.q_heads / s.kv_heads);
  const int nr = rows <= 8 ? 1 : 2;
  SplitPlan p{};
  p.row_tiles = (int)std::min<int64_t>(ceil_div(rows, 8 * nr), 64);
  const int64_t span = plan_span(s, 8 * nr);
  const int64_t items = (int64_t)s.num_seqs * s.kv_heads * p.row_tiles;
  // Turns of the machine.  A few long sequences are cut for one: one of 60000 tokens takes 29 us so, 36 with two,
  // 41 with four.  A batch is ragged and up to four even it out: 19 of up to 8000 take 51, 42, 47 and with eight
  // 58 us, 64 of them 108, 89, 85 and 96.
  const int64_t want = 148 * (nr == 1 ? 4 : 3) * std::min<int64_t>(4, std::max<int64_t>(1, items / 64));
  const int64_t chunks = std::max<int64_t>(1, want / items);
  const int64_t chunk = round_up(std::max<int64_t>(ceil_div(span, chunks), 16 * AT_W), 16 * AT_W);
  // Shorter chunks cost more in the join than they save: 64 sequences of up to 1000 take 23 us in one chunk each and
  // 31 in four, 32 of up to 2000 35 us in chunks of 256 and 26 in 512; where there are few, 256 keep the latency low
  // (one sequence of 2000: 10 us against 12 with 512).
  p.least = items >= 256 ? 1024 : items >= 128 ? 512 : 256;
  p.chunks = (int)std::max<int64_t>(1, ceil_div(span, std::max<int64_t>(chunk, p.least)));
  return p;
}

template <int D, int NR>
void launch_split(const AttendArgs& a, const SplitPlan& p, cudaStream_t st) {
  const dim3 grid((unsigned)(p.chunks * p.row_tiles), (unsigned)a.cache.kv_heads,
                  (unsigned)std::min(a.seq.num_seqs, 65535));
  static OncePerDevice once;
  once([] {
    cudaFuncSetAttribute(attend_split_kernel<D, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, split_smem<D, NR>());
  });
  launch_next(attend_split_kernel<D, NR>, grid, AT_W * 32, split_smem<D, NR>(), st, a, p);
  count_launch();
}

// Eight warps to a row where the rows are few enough for one turn of the machine, or the chunks many.  One sequence of
// 60000 tokens, 74 chunks: 29 us against 35 with one warp; 64 of 8000, 4 chunks: 101 against 96.
template <int D>
void launch_join(const AttendArgs& a, int chunks, cudaStream_t st) {
  const int64_t rows = (int64_t)a.seq.num_tokens * a.q_heads;
  const bool wide = chunks > 4 && (rows <= 1024 || chunks > 16);
  launch_next(wide ? attend_join_kernel<D, 8> : attend_join_kernel<D, 1>, dim3((unsigned)(wide ? rows : ceil_div(rows, 4))),
              wide ? 256 : 128, 0, st, a, chunks);
  count_launch();
}

struct AttendPlan {
  bool tc;
  int chunks;
  SplitPlan split;
};

// Which kernel.  Per key of a sequence and key head the split kernel takes 30 ps and 30 more for each tile of 16 rows;
// the tensor-core kernel 2.4 us for 128 keys and 256 rows on each of 148 processors.  Where its blocks leave
// processors idle it gets chunks of the keys, of 256 at least (one sequence of 2000, 64 new tokens: 25 us, 29 with 512;
// of 60000, 1280 tokens, 160 blocks: 2234 us whole, 1398 in eight; of 2000: 73 whole, 102 in two).
// Both sides, split and tensor core, 4 query heads on each of 8 key heads, us:
//   new tokens                4          12         16         32         64         500
//   1 sequence of 60000    37   80    74   81    96   82   186   86   351   93   2467  581
//   1 of 2000              14   19    17   21    17   21    23   23    33   25    132   45
//   16 of up to 8000       61  162   118  163   147  162   249  164   419  165   2920  741
//   64 of up to 4000       90  220   180  223   228  223   410  224   775  230   5432 1368
AttendPlan attend_plan(const AttendShape& s) {
  const int64_t rows = (int64_t)s.max_q * (s.q_heads / s.kv_heads), heads = (int64_t)s.num_seqs * s.kv_heads;
  const int64_t span = plan_span(s, 256), steps = ceil_div(span, 128), blocks = heads * ceil_div(rows, 256);
  // A turn of blocks takes 12 us beside its steps; chunks 5 us for the join and 2.5 ps for each of the D values that a
  // row of a chunk writes and the join reads.  Several sequences are ragged, which evens out their turns: they are cut
  // for one turn at most.
  const int64_t rows_all = std::min<int64_t>(s.num_tokens, (int64_t)s.num_seqs * s.max_q) * s.q_heads;
  int64_t chunks = 1;
  double tc = 0.0, least = 1e30;
  for (int64_t t = 0; t <= (s.num_seqs > 1 ? 1 : 16); ++t) {  // whole, or as many chunks as t turns hold
    int64_t c = std::min<int64_t>(148 * t / blocks, steps / 2);
    c = c > 1 ? ceil_div(steps, ceil_div(steps, c)) : 1;
    const int64_t turns = ceil_div(blocks * c, 148);
    const double work = 2.4 * (double)(turns * ceil_div(steps, c));
    const double all = work + 12.0 * (double)turns + (c > 1 ? 5.0 + 2.5e-6 * (double)(rows_all * s.D * c) : 0.0);
    if (all < least) chunks = c, tc = work, least = all;
  }
  const double split = 30e-6 * (double)heads * (double)span * (double)(1 + ceil_div(rows, 16));
  AttendPlan p{tc < split, (int)chunks, {}};
  // hints may be far off: the workspace stays below half a gigabyte
  const int64_t most = std::max<int64_t>(1, (int64_t(1) << 29) / (4 * std::max<int64_t>(1, (int64_t)s.num_tokens * s.q_heads) * (s.D + 2)));
  if (!p.tc) p.split = split_plan(s), p.chunks = p.split.chunks;
  p.chunks = p.split.chunks = (int)std::min<int64_t>(p.chunks, most);
  return p;
}

}  // namespace

size_t attend_workspace(const AttendShape& s) {
  const int chunks = attend_plan(s).chunks;
  if (chunks == 1) return 0;
  const int64_t rows = (int64_t)chunks * s.num_tokens * s.q_heads;
  return (size_t)(round_up(rows * 2, 4) + rows * s.D) * 4;
}

void launch_attend(const AttendArgs& a, const AttendShape& s, cudaStream_t st) {
  const AttendPlan p = attend_plan(s);
  if (p.tc) {
    launch_attend_tc(a, s, p.chunks, st);
  } else {
    const bool one = (int64_t)s.max_q * (s.q_heads / s.kv_heads) <= 8;
    if (s.D == 128) one ? launch_split<128, 1>(a, p.split, st) : launch_split<128, 2>(a, p.split, st);
    else one ? launch_split<64, 1>(a, p.split, st) : launch_split<64, 2>(a, p.split, st);
  }
  if (p.chunks > 1) s.D == 128 ? launch_join<128>(a, p.chunks, st) : launch_join<64>(a, p.chunks, st);
}

}  // namespace kl
