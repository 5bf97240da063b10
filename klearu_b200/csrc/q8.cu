// q8.cu -- 8-bit rows and their products.
//
//  * rows of 8-bit codes with one f32 scale each, x ~ scale * code with
//    scale = max|x| / 127, from a row as it is or from its root-mean-square
//    norm after a residual addition (the norm of klearu-llm's model/
//    rms_norm.rs, which kl_ffn_stack_decode applies in f32);
//  * out = (A . W^T) * sa * sw (+ bias) (+ out), A and W such codes, the
//    products summed as 32-bit integers, so the sum is exact in any order.
#include <algorithm>

#include "engine.h"
#include "pdl.cuh"
#include "tcgen05.cuh"

namespace kl {
namespace {

__device__ __forceinline__ bool finite32(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

__device__ __forceinline__ float norm_weight(const NormQ8Args& a, int c) {
  return a.weight ? (a.one_plus ? 1.f + a.weight[c] : a.weight[c]) : 1.f;
}
__device__ __forceinline__ void norm_weights8(const NormQ8Args& a, int c, float* w) {
  if (!a.weight) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.f;
    return;
  }
  *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(a.weight + c);
  *reinterpret_cast<float4*>(w + 4) = *reinterpret_cast<const float4*>(a.weight + c + 4);
  if (a.one_plus) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.f + w[i];
  }
}
// rint(127 u / top) for u = h * w in 64 bits.  The f32 quotient decides unless
// it is within 1e-4 of a border between two codes (its own error is below
// 3 roundings of 127, 2.3e-5): only then are the 64-bit product and quotient
// taken, so the codes are those of the definition.  Where the row's largest is so
// small that 127 / top is no f32 (below 3.7e-37), every code is taken so.
__device__ __noinline__ int q8_exact(float h, float w, double top) {
  return (int)rint((double)h * (double)w * 127.0 / top);
}
// Where eps is too small to matter beside them: squares of values below 2^-40, many of which are no normal numbers, are
// summed once more times 2^200.
__host__ __device__ __forceinline__ bool q8_small_eps(const NormQ8Args& a) { return a.norm && a.eps < 0x1p-75f; }
__device__ __forceinline__ bool q8_small(const NormQ8Args& a, float ss) { return q8_small_eps(a) && ss < 0x1p-80f; }
// A row's scale.  mx, the largest product in f32, has lost bits where it is among the smallest numbers; top has not.
__device__ __forceinline__ float q8_scale(const NormQ8Args& a, float mx, double top, float ss, bool small) {
  if (small) return (float)(top * (0x1p100 / 127.0) * (double)(1.f / sqrtf(ss / (float)a.cols + a.eps * 0x1p100f * 0x1p100f)));
  const float rinv = a.norm ? 1.f / sqrtf(ss / (float)a.cols + a.eps) : 1.f;
  return mx < 1e-30f ? (float)(top * (1.0 / 127.0) * (double)rinv) : mx * rinv / 127.f;
}
__device__ __forceinline__ int q8_code(float h, float w, float p, float inv, double top) {
  const float t = p * inv;
  const float r = rintf(t);
  if (!(fabsf(fabsf(t - r) - 0.5f) >= 1e-4f)) return q8_exact(h, w, top);  // NaN where inv is infinite
  return (int)r;
}

template <int NT>
__device__ __forceinline__ float block_reduce(float v, float* tmp, bool is_max) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(FULL, v, o);
    v = is_max ? fmaxf(v, u) : v + u;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = tmp[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) v = is_max ? fmaxf(v, tmp[i]) : v + tmp[i];
  return v;
}

// One block per row, a row's 8 NV blockDim values in registers, 16 bytes and
// more a load; one pass over memory.  8191 rows of 4096 bf16 columns and their
// residual: 79 us, 4.7 TB/s; bound by each block's chain of load, two barriers
// and store.  Resident blocks that fetch their next row meanwhile took 91.
// SMALL: eps may be too small for the squares of small rows; keeping h for that
// costs registers (201 us with the values formed after it, 199 without).
template <int NV, class T, bool SMALL>
__global__ void __launch_bounds__(1024) norm_q8_vec_kernel(NormQ8Args a) {
  __shared__ float2 tmp[32];
  __shared__ unsigned long long top_s;
  begin_next();
  after_before();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const float* r = a.residual ? a.residual + row * a.ldr : nullptr;
  float* ho = a.hidden ? a.hidden + row * a.ldh : nullptr;
  float h[NV][8], p[NV][8], ss = 0.f, mx = 0.f, z = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * blockDim.x + threadIdx.x) * 8;
    if (c < a.cols) {
      if (sizeof(T) == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(x + c);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h[v][2 * i] = __uint_as_float(w[i] << 16);
          h[v][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      } else {
        *reinterpret_cast<float4*>(&h[v][0]) = *reinterpret_cast<const float4*>(x + c);
        *reinterpret_cast<float4*>(&h[v][4]) = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + c + 4);
      }
      if (r) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 y = *reinterpret_cast<const float4*>(r + c + i);
          h[v][i] += y.x;
          h[v][i + 1] += y.y;
          h[v][i + 2] += y.z;
          h[v][i + 3] += y.w;
        }
      }
      if (ho) {
        *reinterpret_cast<float4*>(ho + c) = make_float4(h[v][0], h[v][1], h[v][2], h[v][3]);
        *reinterpret_cast<float4*>(ho + c + 4) = make_float4(h[v][4], h[v][5], h[v][6], h[v][7]);
      }
      float w8[8];
      norm_weights8(a, c, w8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[v][i] = h[v][i] * w8[i];
        z = fmaf(p[v][i], 0.f, z);  // NaN for a product that is not finite, as it is for such an h
        ss = fmaf(h[v][i], h[v][i], ss);
        mx = fmaxf(mx, fabsf(p[v][i]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[v][i] = p[v][i] = 0.f;
    }
  }
  const float most = mx;  // of this thread
  if (z != 0.f) mx = INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(FULL, ss, o);
    mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
  }
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = make_float2(ss, mx);
  if (threadIdx.x == 0) top_s = 0ull;
  __syncthreads();
  const float2 of = (int)(threadIdx.x & 31) < warps ? tmp[threadIdx.x & 31] : make_float2(0.f, 0.f);
  ss = of.x;
  mx = of.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(FULL, ss, o);
    mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
  }
  // the largest |h w| in 64 bits is among those whose f32 product is largest
  if (most == mx) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * blockDim.x + threadIdx.x) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (fabsf(p[v][i]) == mx && c < a.cols)
          atomicMax(&top_s, (unsigned long long)__double_as_longlong(fabs((double)h[v][i] * (double)norm_weight(a, c + i))));
    }
  }
  __syncthreads();
  const unsigned long long top_bits = top_s;
  const double top = __longlong_as_double((long long)top_bits);
  const bool good = finite32(mx) && (!a.norm || finite32(ss));
  auto put_scale = [&](bool small) {
    if (threadIdx.x == 0) a.scales[row] = good ? q8_scale(a, mx, top, ss, small) : __int_as_float(0x7fffffff);
  };
  if (!SMALL) put_scale(false);
  const float inv = good && top_bits ? 127.f / mx : 0.f;  // infinite where the products are too small for f32
  int8_t* co = a.codes + row * a.ldc;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * blockDim.x + threadIdx.x) * 8;
    if (c >= a.cols) continue;
    uint32_t out[2] = {0, 0};
    if (inv > 0.f) {
      uint32_t b[8];
      float off = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float t = p[v][i] * inv, y = t + 12582912.f;  // 1.5 * 2^23: rounds to a whole number, in the low bits
        off = fmaxf(off, fabsf(t - (y - 12582912.f)));
        b[i] = __float_as_uint(y);
      }
      if (off > 0.4999f || inv == INFINITY) {  // a border between two codes is near
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!(fabsf(p[v][i] * inv - (__uint_as_float(b[i]) - 12582912.f)) <= 0.4999f))
            b[i] = (uint32_t)q8_exact(h[v][i], norm_weight(a, c + i), top);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        out[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
    }
    *reinterpret_cast<uint2*>(co + c) = make_uint2(out[0], out[1]);
  }
  if (!SMALL) return;
  const bool small = q8_small(a, ss);
  if (small) {
    ss = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(h[v][i] * 0x1p100f, h[v][i] * 0x1p100f, ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
    if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5].x = ss;
    __syncthreads();
    ss = (int)(threadIdx.x & 31) < warps ? tmp[threadIdx.x & 31].x : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
  }
  put_scale(small);
}

// The same for any alignment and width: the row's h waits in shared memory
// between the pass that finds its sum of squares and maximum and the pass that
// writes the codes.
template <int NT, class T>
__global__ void __launch_bounds__(NT) norm_q8_kernel(NormQ8Args a) {
  extern __shared__ float nq_h[];
  __shared__ float tmp[NT / 32];
  __shared__ unsigned long long top_s;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const float* r = a.residual ? a.residual + row * a.ldr : nullptr;
  float* ho = a.hidden ? a.hidden + row * a.ldh : nullptr;
  begin_next();
  after_before();
  if (threadIdx.x == 0) top_s = 0ull;
  float ss = 0.f, mx = 0.f;
  bool fin = true;
  for (int i = threadIdx.x; i < a.cols; i += NT) {
    float h = to_f(x[i]);
    if (r) h += r[i];
    if (ho) ho[i] = h;
    nq_h[i] = h;
    const float w = norm_weight(a, i);
    const float p = h * w;
    fin = fin && finite32(p) && finite32(h);
    ss = fmaf(h, h, ss);
    mx = fmaxf(mx, fabsf(p));
  }
  ss = block_reduce<NT>(ss, tmp, false);
  mx = block_reduce<NT>(fin ? mx : INFINITY, tmp, true);
  // the largest |h w| in 64 bits is among those whose f32 product is largest
  for (int i = threadIdx.x; i < a.cols; i += NT) {
    const float w = norm_weight(a, i);
    if (fabsf(nq_h[i] * w) == mx)
      atomicMax(&top_s, (unsigned long long)__double_as_longlong(fabs((double)nq_h[i] * (double)w)));
  }
  __syncthreads();
  const unsigned long long top_bits = top_s;
  const double top = __longlong_as_double((long long)top_bits);
  const bool good = finite32(mx) && (!a.norm || finite32(ss)), small = q8_small(a, ss);
  if (small) {
    ss = 0.f;
    for (int i = threadIdx.x; i < a.cols; i += NT) ss = fmaf(nq_h[i] * 0x1p100f, nq_h[i] * 0x1p100f, ss);
    ss = block_reduce<NT>(ss, tmp, false);
  }
  if (threadIdx.x == 0) a.scales[row] = good ? q8_scale(a, mx, top, ss, small) : __int_as_float(0x7fffffff);
  const float inv = good && top_bits ? 127.f / mx : 0.f;  // infinite where the products are too small for f32
  int8_t* co = a.codes + row * a.ldc;
  for (int i = threadIdx.x; i < a.cols; i += NT) {
    const float w = norm_weight(a, i);
    co[i] = inv > 0.f ? (int8_t)q8_code(nq_h[i], w, nq_h[i] * w, inv, top) : (int8_t)0;
  }
}

// ---- the product ----
// The weights are kept as tiles of 128 channels by 128 bytes of K, each 16 KB
// contiguous and in the swizzled order that the tensor core reads (chunk e of 16
// bytes of channel r at e ^ (r & 7)), so that one untiled copy brings a tile:
// fetched as boxes out of rows 4 KB apart they came at 40 bytes a ns and SM.
// out^T in tiles: 128 output channels (rows of W: the MMA's M) by nt rows of A
// (its N), so that the weights, the larger operand of a decode step, fill the
// 128 lanes whatever the number of rows, and a warp's stores of one row of out
// are 32 neighbouring channels.  A arrives by TMA in boxes of 128 bytes of K
// (128-byte swizzle); four MMAs of K = 32 to a chunk; rows and K beyond the
// matrices are zeros.
constexpr int Q8_KB = 128;               // bytes of K per stage
constexpr int Q8_WTILE = 128 * Q8_KB;    // weight bytes of a stage

struct Q8Tile {
  int nt;      // rows of A per tile, a multiple of 16
  int stages;
  int kc;      // K chunks of 128
  uint32_t tmem_cols;
  int join;  // rows that a block of a split finishes, a multiple of 4
};

enum Q8Out { Q8_F32, Q8_BF16, Q8_ADD };  // add: to an f32 out
__device__ __forceinline__ float q8_value(int acc, float sa, float sw, float bias) {
  return fmaf((float)acc * sa, sw, bias);
}
template <int OUT>
__device__ __forceinline__ void q8_put(char* p, float v) {
  if (OUT == Q8_BF16) *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(v);
  else if (OUT == Q8_F32) *reinterpret_cast<float*>(p) = v;
  else *reinterpret_cast<float*>(p) += v;
}
template <int OUT>
__device__ __forceinline__ char* q8_at(const Q8Args& a, int64_t r, int64_t c) {
  return static_cast<char*>(a.out) + (r * a.ldo + c) * (OUT == Q8_BF16 ? 2 : 4);
}
// Rows [0, rows) of a tile from the thread's lane of tensor memory to channel c
// of out; sa: the rows' scales.  The warp takes part as one; live: c is a channel.
template <int OUT>
__device__ __forceinline__ void q8_rows(const Q8Args& a, uint32_t taddr, int64_t row, int rows, int64_t c, bool live,
                                        const float* sa, float sw, float bias) {
  char* p = q8_at<OUT>(a, row, c);
  const int64_t step = a.ldo * (OUT == Q8_BF16 ? 2 : 4);
#pragma unroll 1
  for (int j = 0; j < rows; j += 16) {
    uint32_t v[16];
    float s[16];
    tc5_ld16_async(taddr + j, v);
#pragma unroll
    for (int u = 0; u < 16; u += 4) *reinterpret_cast<float4*>(s + u) = *reinterpret_cast<const float4*>(sa + j + u);
    tc5_ld_wait();
    if (live && j + 16 <= rows) {
#pragma unroll
      for (int u = 0; u < 16; ++u, p += step) q8_put<OUT>(p, q8_value((int)v[u], s[u], sw, bias));
    } else if (live) {
#pragma unroll
      for (int u = 0; u < 16; ++u, p += step)
        if (j + u < rows) q8_put<OUT>(p, q8_value((int)v[u], s[u], sw, bias));
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void st_cluster4(uint32_t saddr, uint32_t rank, const uint32_t* v) {
  uint32_t p;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(p) : "r"(saddr), "r"(rank));
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

// Where a ring stands: its stage, and how often it has been round.  Counted, not
// divided out: these loops are one thread's, and two divisions a chunk of K made
// a chunk 800 cycles long.
struct Q8Ring {
  int stage = 0;
  uint32_t round = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) {
      stage = 0;
      ++round;
    }
  }
};
// One chunk of K of a tile: its weights, announcing both, and its rows.
__device__ __forceinline__ void q8_load_w(const int8_t* tile, const Q8Tile& t, unsigned char* sm, uint64_t* full, int stage) {
  const int size = Q8_WTILE + t.nt * Q8_KB;
  mbar_arrive_expect_tx(full + stage, (uint32_t)size);
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(sm + stage * size)),
      "l"(tile), "r"(Q8_WTILE), "r"(smem_u32(full + stage))
      : "memory");
}
__device__ __forceinline__ void q8_load_a(const CUtensorMap* am, const Q8Tile& t, unsigned char* sm, uint64_t* full, int c,
                                          int row, int stage) {
  tma_load_2d(sm + stage * (Q8_WTILE + t.nt * Q8_KB) + Q8_WTILE, am, c * Q8_KB, row, full + stage);
}
// The loading side of a tile: K chunks [c0, c1) through the ring.  False when a
// wait gave up.
__device__ __forceinline__ bool q8_load(const int8_t* w, const CUtensorMap* am, const Q8Tile& t, unsigned char* sm,
                                        uint64_t* full, uint64_t* empty, int ch, int row, int c0, int c1, Q8Ring& q) {
  const int8_t* tile = w + ((int64_t)(ch >> 7) * t.kc + c0) * Q8_WTILE;
  for (int c = c0; c < c1; ++c, q.next(t.stages), tile += Q8_WTILE) {
    if (q.round > 0 && !mbar_wait(&empty[q.stage], (q.round - 1) & 1u)) return false;
    q8_load_w(tile, t, sm, full, q.stage);
    q8_load_a(am, t, sm, full, c, row, q.stage);
  }
  return true;
}
__device__ __forceinline__ bool q8_mma(const Q8Tile& t, unsigned char* sm, uint64_t* full, uint64_t* empty, uint32_t tmem,
                                       int chunks, Q8Ring& q) {
  const uint32_t idesc = i8_idesc(128, t.nt), size = (uint32_t)(Q8_WTILE + t.nt * Q8_KB) >> 4;
  const uint64_t d0 = sw128_desc(smem_u32(sm));
  for (int c = 0; c < chunks; ++c, q.next(t.stages)) {
    if (!mbar_wait(&full[q.stage], q.round & 1u)) return false;
    tc5_fence_after();
    const uint64_t dw = d0 + (uint64_t)(q.stage * size), da = dw + (Q8_WTILE >> 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) tc5_mma_i8(tmem, dw + 2 * k, da + 2 * k, idesc, (c | k) != 0);
    tc5_commit(&empty[q.stage]);
  }
  return true;
}
// No copy may be in flight when the block ends: the last round of every stage.
__device__ __forceinline__ void q8_drain(const Q8Tile& t, uint64_t* full, const Q8Ring& q) {
  for (int s = 0; s < t.stages; ++s) {
    const uint32_t rounds = q.round + (s < q.stage ? 1 : 0);
    if (rounds > 0) mbar_wait(&full[s], (rounds - 1) & 1u);
  }
}

// Few tiles: one tile per cluster, its K split over the cluster's blocks; each
// block finishes a share of the tile's rows, for which the others store their
// 32-bit sums in its shared memory (whole numbers: any order gives the same
// sum).  One launch, no workspace.
template <int OUT>
__global__ void __launch_bounds__(128) q8_split_kernel(const __grid_constant__ CUtensorMap am, Q8Args a, Q8Tile t,
                                                       int splits) {
  extern __shared__ unsigned char q8_dyn[];
  __shared__ uint64_t full[12], empty[12], done;
  __shared__ uint32_t tmem_s;
  __shared__ int fail;
  __shared__ __align__(16) float sa[256];  // the tile's row scales: read between stores to out, they must not wait for memory
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(q8_dyn) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = splits > 1 ? (int)cluster_rank() : 0;
  const int ch = (blockIdx.x / splits) * 128, row = blockIdx.y * t.nt;
  const int c0 = (int)((int64_t)t.kc * rank / splits), c1 = (int)((int64_t)t.kc * (rank + 1) / splits);
  const int c = ch + threadIdx.x, first = min(c0 + t.stages, c1);
  int* part = reinterpret_cast<int*>(sm + t.stages * (Q8_WTILE + t.nt * Q8_KB));  // of a split: behind the ring
  Q8Ring q;  // of chunks loaded, or multiplied
  if (splits > 1) cluster_arrive();
  if (threadIdx.x == 0) {
    prefetch_map(&am);
    for (int s = 0; s < t.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    fail = 0;
    fence_mbar_init();
    // the ring's first fills go out before anything else is ready, the weights before the rows are
    const int8_t* tile = a.w + ((int64_t)(ch >> 7) * t.kc + c0) * Q8_WTILE;
    for (int i = c0; i < first; ++i, tile += Q8_WTILE) q8_load_w(tile, t, sm, full, i - c0);
    after_before();
    for (int i = c0; i < first; ++i, q.next(t.stages)) q8_load_a(&am, t, sm, full, i, row, q.stage);
  }
  // what the end needs, while the ring fills
  const float sw = c < a.n ? a.w_scale[c] : 0.f, bias = a.bias && c < a.n ? a.bias[c] : 0.f;
  after_before();
  for (int j = threadIdx.x; j < t.nt; j += 128) sa[j] = row + j < a.m ? a.a_scale[row + j] : 0.f;
  if (warp == 1) tc5_alloc(&tmem_s, t.tmem_cols);
  tc5_fence_before();
  __syncthreads();
  tc5_fence_after();
  begin_next();  // not before this block has its tensor memory, which the next one's may wait for
  const uint32_t tmem = tmem_s;
  if (warp == 0 && lane == 0) {
    if (!q8_load(a.w, &am, t, sm, full, empty, ch, row, first, c1, q)) atomicExch(&fail, 1);
    q8_drain(t, full, q);
  } else if (warp == 1 && lane == 0) {
    if (!q8_mma(t, sm, full, empty, tmem, c1 - c0, q)) atomicExch(&fail, 1);
    tc5_commit(&done);
    if (!mbar_wait(&done, 0)) atomicExch(&fail, 1);
  }
  __syncthreads();
  tc5_fence_after();
  const uint32_t mine = tmem + ((uint32_t)warp << 21);  // lane 32 * warp
  const int rows = min(t.nt, a.m - row);
  if (splits == 1) {
    q8_rows<OUT>(a, mine, row, rows, c, c < a.n, sa, sw, bias);
  } else {
    // Block r finishes rows [r each, (r + 1) each), for which each block stores its sums there, [from][channel][row].
    const int each = t.join;
    cluster_wait();  // all blocks have begun, their shared memory is there
    const uint32_t at = smem_u32(part + (rank * 128 + (int)threadIdx.x) * each);
    int to = 0, off = 0;  // whose rows these are, and where in its share
#pragma unroll 1
    for (int j = 0; j < rows; j += 16) {
      uint32_t v[16];
      tc5_ld16_async(mine + j, v);
      tc5_ld_wait();
#pragma unroll
      for (int u = 0; u < 16; u += 4) {
        if (j + u < rows) st_cluster4(at + 4 * (uint32_t)off, (uint32_t)to, v + u);
        if ((off += 4) == each) {
          off = 0;
          ++to;
        }
      }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const int from = rank * each, end = min(from + each, rows);
#pragma unroll 2
    for (int j = from; j < end; j += 4) {
      int s[4] = {0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r < splits) {
          const int4 v = *reinterpret_cast<const int4*>(part + (r * 128 + (int)threadIdx.x) * each + j - from);
          s[0] += v.x;
          s[1] += v.y;
          s[2] += v.z;
          s[3] += v.w;
        }
      }
      char* p = q8_at<OUT>(a, row + j, c);
#pragma unroll
      for (int u = 0; u < 4; ++u, p += a.ldo * (OUT == Q8_BF16 ? 2 : 4))
        if (c < a.n && j + u < end) q8_put<OUT>(p, q8_value(s[u], sa[j + u], sw, bias));
    }
  }
  tc5_fence_before();
  __syncthreads();
  if (fail && threadIdx.x == 0) atomicOr(a.err, DERR_TIMEOUT);
  if (warp == 1) tc5_dealloc(tmem, t.tmem_cols);
}

// Many tiles: one block per SM takes tiles in turn, two accumulators in tensor
// memory so that the tile before is written while the next one multiplies.
constexpr int Q8_PN = 256;
constexpr int Q8_PNT = 320;  // 10 warps: loads, MMAs, 8 that write, two to a quarter of the lanes
template <int OUT>
__global__ void __launch_bounds__(Q8_PNT, 1) q8_persistent_kernel(const __grid_constant__ CUtensorMap am, Q8Args a,
                                                                  Q8Tile t, int ch_tiles, int tiles) {
  extern __shared__ unsigned char q8_dyn[];
  __shared__ uint64_t full[12], empty[12], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_s;
  __shared__ int fail;
  __shared__ __align__(16) float sa[8][Q8_PN / 2];  // each writing warp's copy of its half of the tile's row scales
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(q8_dyn) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < t.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);
    }
    fail = 0;
    fence_mbar_init();
  }
  if (warp == 1) tc5_alloc(&tmem_s, 512);
  tc5_fence_before();
  __syncthreads();
  tc5_fence_after();
  const uint32_t tmem = tmem_s;
  volatile int* vf = &fail;
  if (warp == 0) {
    if (lane == 0) {
      Q8Ring q;
      for (int i = blockIdx.x; i < tiles; i += gridDim.x)
        if (*vf || !q8_load(a.w, &am, t, sm, full, empty, i % ch_tiles * 128, i / ch_tiles * Q8_PN, 0, t.kc, q)) {
          atomicExch(&fail, 1);
          break;
        }
      q8_drain(t, full, q);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      Q8Ring q;
      int n = 0;
      for (int i = blockIdx.x; i < tiles; i += gridDim.x, ++n) {
        const int b = n & 1;
        if ((n >= 2 && !mbar_wait(&acc_empty[b], (uint32_t)(n / 2 - 1) & 1u)) ||
            (tc5_fence_after(), *vf || !q8_mma(t, sm, full, empty, tmem + b * Q8_PN, t.kc, q))) {
          atomicExch(&fail, 1);
          break;
        }
        tc5_commit(&acc_full[b]);
      }
    }
  } else {
    const int quad = warp & 3;  // the tensor-memory lanes that this warp may read
    const int half = (warp - 2) >> 2;
    float* scale = sa[warp - 2];
    int n = 0;
    for (int i = blockIdx.x; i < tiles; i += gridDim.x, ++n) {
      const int b = n & 1;
      const int c = i % ch_tiles * 128 + quad * 32 + lane, row = i / ch_tiles * Q8_PN + half * (Q8_PN / 2);
      const int rows = max(0, min(Q8_PN / 2, a.m - row));
      const float sw = c < a.n ? a.w_scale[c] : 0.f, bias = a.bias && c < a.n ? a.bias[c] : 0.f;
      __syncwarp();
      for (int j = lane; j < Q8_PN / 2; j += 32) scale[j] = row + j < a.m ? a.a_scale[row + j] : 0.f;
      __syncwarp();
      if (__any_sync(FULL, *vf || !mbar_wait(&acc_full[b], (uint32_t)(n / 2) & 1u))) {
        atomicExch(&fail, 1);
        break;
      }
      tc5_fence_after();
      q8_rows<OUT>(a, tmem + ((uint32_t)quad << 21) + b * Q8_PN + half * (Q8_PN / 2), row, rows, c, c < a.n, scale, sw, bias);
      tc5_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[b]);
    }
  }
  tc5_fence_before();
  __syncthreads();
  if (fail && threadIdx.x == 0) atomicOr(a.err, DERR_TIMEOUT);
  if (warp == 1) tc5_dealloc(tmem, 512);
}

int q8_sms() {
  static int n = [] {
    int dev = 0, v = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    return v;
  }();
  return n;
}

// One or two rows: every warp streams pairs of channels' weights, four 16-byte
// loads of each in flight per lane, against the rows in shared memory, four
// products an instruction.  No ring, tensor memory or join to set up: with one
// row and 50 MB of weights that is 5 of 16 us.
constexpr int Q8_VW = 4;  // warps per block
template <int OUT, int M>
__global__ void __launch_bounds__(Q8_VW * 32) q8_vector_kernel(Q8Args a) {
  extern __shared__ __align__(16) int8_t q8_rows[];  // [M][128 kc], zero from k on as the weights are
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = (blockIdx.x * Q8_VW + warp) * 2;
  const int words = (a.k + Q8_KB - 1) / Q8_KB * 8;  // of 16 bytes
  const int8_t* tile = a.w + (int64_t)(c0 >> 7) * (words >> 3) * Q8_WTILE + (c0 & 127) * Q8_KB;  // c0 is even
  const int s0 = c0 & 7;
  uint4 x[2][4];
  auto load = [&](int at) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = at + u * 32 + lane;
      const int8_t* p = tile + (int64_t)(i >> 3) * Q8_WTILE;
      const bool in = i < words && c0 < a.n;
      x[0][u] = in ? __ldcs(reinterpret_cast<const uint4*>(p + (((i & 7) ^ s0) << 4))) : make_uint4(0, 0, 0, 0);
      x[1][u] = in ? __ldcs(reinterpret_cast<const uint4*>(p + Q8_KB + (((i & 7) ^ (s0 + 1)) << 4))) : make_uint4(0, 0, 0, 0);
    }
  };
  begin_next();
  load(0);  // the first weights on their way while the rows are staged
  after_before();
  for (int i = threadIdx.x; i < M * words; i += Q8_VW * 32) {
    const int r = i / words, at = (i - r * words) * 16;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (at + 16 <= a.k) {
      v = *reinterpret_cast<const uint4*>(a.a + r * a.lda + at);
    } else if (at < a.k) {
      uint32_t b[4] = {0, 0, 0, 0};
      for (int e = 0; at + e < a.k; ++e) b[e >> 2] |= (uint32_t)(uint8_t)a.a[r * a.lda + at + e] << (8 * (e & 3));
      v = make_uint4(b[0], b[1], b[2], b[3]);
    }
    reinterpret_cast<uint4*>(q8_rows)[i] = v;
  }
  __syncthreads();
  int acc[M][2] = {};
  for (int at = 0; at < words; at += 128) {
    if (at > 0) load(at);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = min(at + u * 32 + lane, words - 1);  // beyond the end the weights are zero
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const uint4 y = reinterpret_cast<const uint4*>(q8_rows)[m * words + i];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          acc[m][c] = __dp4a((int)x[c][u].x, (int)y.x, acc[m][c]);
          acc[m][c] = __dp4a((int)x[c][u].y, (int)y.y, acc[m][c]);
          acc[m][c] = __dp4a((int)x[c][u].z, (int)y.z, acc[m][c]);
          acc[m][c] = __dp4a((int)x[c][u].w, (int)y.w, acc[m][c]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int sum = warp_sum(acc[m][c]);
      if (lane == 0 && c0 + c < a.n)
        q8_put<OUT>(q8_at<OUT>(a, m, c0 + c), q8_value(sum, a.a_scale[m], a.w_scale[c0 + c], a.bias ? a.bias[c0 + c] : 0.f));
    }
}

__global__ void q8_pack_kernel(const int8_t* src, int64_t ld, int n, int k, int kc, int8_t* dst) {
  const int p = blockIdx.x * blockDim.x + threadIdx.x;  // 16 bytes of K
  const int64_t r = (int64_t)blockIdx.z * 65535 + blockIdx.y;
  if (p >= kc * 8 || r >= round_up(n, 128)) return;
  uint32_t b[4] = {0, 0, 0, 0};
  if (r < n)
    for (int e = 0; e < 16 && p * 16 + e < k; ++e) b[e >> 2] |= (uint32_t)(uint8_t)src[r * ld + p * 16 + e] << (8 * (e & 3));
  *reinterpret_cast<uint4*>(dst + ((r >> 7) * kc + (p >> 3)) * Q8_WTILE + (r & 127) * Q8_KB + (((p & 7) ^ (int)(r & 7)) << 4)) =
      make_uint4(b[0], b[1], b[2], b[3]);
}

}  // namespace

// Vectors where the weights and every row start on 16 bytes (codes 8) and cols is a multiple of
// 8 up to 16384: 8 values a thread while the rows do not fill the machine, 16
// where they do (fewer threads to wait for at the two barriers).
static bool norm_vec(const NormQ8Args& a) {
  auto on = [](const void* p, int64_t ld, int size, int to) {
    return !p || (reinterpret_cast<uintptr_t>(p) % to == 0 && ld * size % to == 0);
  };
  return a.cols % 8 == 0 && a.cols <= 16384 && on(a.x, a.ldx, a.x_bf16 ? 2 : 4, 16) && on(a.residual, a.ldr, 4, 16) &&
         on(a.hidden, a.ldh, 4, 16) && on(a.codes, a.ldc, 1, 8) && on(a.weight, 0, 4, 16);
}
void launch_norm_q8(const NormQ8Args& a, int rows, cudaStream_t st) {
  if (norm_vec(a)) {
    // Eight values a thread while the rows are two blocks a processor at most, then sixteen, half the threads (4096 bf16
    // columns, us, with the values formed after it): 148 rows 10.4 against 12.4, 400 18.6 and 16.6, 8191 221 and 205.
    // The plain kernel takes 14.5, 21.2 and 247: rows that are not aligned, and more than 16384 columns.
    const bool two = a.cols > 8192 || rows > 296;
    const int threads = (int)round_up(ceil_div(a.cols, two ? 16 : 8), 32);
    auto pick = [&](auto small) {
      constexpr bool S = decltype(small)::value;
      return a.x_bf16 ? two ? norm_q8_vec_kernel<2, __nv_bfloat16, S> : norm_q8_vec_kernel<1, __nv_bfloat16, S>
                      : two ? norm_q8_vec_kernel<2, float, S> : norm_q8_vec_kernel<1, float, S>;
    };
    auto* kernel = q8_small_eps(a) ? pick(std::true_type{}) : pick(std::false_type{});
    launch_next(kernel, dim3(rows), threads, 0, st, a);
    count_launch();
    return;
  }
  static OncePerDevice once;
  once([] {
    cudaFuncSetAttribute(norm_q8_kernel<256, float>, cudaFuncAttributeMaxDynamicSharedMemorySize, NORM_Q8_MAX_COLS * 4);
    cudaFuncSetAttribute(norm_q8_kernel<256, __nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         NORM_Q8_MAX_COLS * 4);
  });
  const size_t sm = (size_t)a.cols * 4;
  launch_next(a.x_bf16 ? norm_q8_kernel<256, __nv_bfloat16> : norm_q8_kernel<256, float>, dim3(rows), 256, sm, st, a);
  count_launch();
}

size_t q8_weight_bytes(int n, int k) { return (size_t)ceil_div(n, 128) * ceil_div(k, Q8_KB) * Q8_WTILE; }
void launch_q8_pack(const int8_t* src, int64_t ld, int n, int k, int8_t* dst, cudaStream_t st) {
  const int kc = (int)ceil_div(k, Q8_KB);
  const int64_t rows = round_up(n, 128);
  q8_pack_kernel<<<dim3((unsigned)ceil_div(kc * 8, 128), (unsigned)std::min<int64_t>(rows, 65535),
                        (unsigned)ceil_div(rows, 65535)),
                   128, 0, st>>>(src, ld, n, k, kc, dst);
  count_launch();
}

// Rows per tile and splits of K, by what was measured: a block takes 0.3 us and
// 0.25 ns a row of its tile for a chunk of 128 bytes of K (one thread's loop), two
// blocks share an SM up to 64 rows; the weights take 6.2 bytes a ns from memory
// and 12 where other tiles of rows read them again; 2 us a further turn of blocks,
// 3 us to join a split.  Splits that the weights' stream bounds are priced alike,
// and the fewest are taken (33 x 4096 of 11008: 4 of 4 to 8; others within 5%).
// More tiles of 256 rows than SMs: the persistent kernel
// (us, persistent and not; k 4096: 300 x 12288 30.6 33.8, 513 x 12288 32.9 39.2,
// 1000 x 4096, 128 tiles, 20.6 20.7, 2000 x 4096 32.3 39.0).
struct Q8Plan {
  bool persistent;
  int nt, splits;
};
static Q8Plan q8_plan(const Q8Args& a) {
  const int sms = q8_sms();
  const int64_t ch = ceil_div(a.n, 128), kc = ceil_div(a.k, Q8_KB);
  const int most = (int)std::min<int64_t>(256, round_up(a.m, 16));
  if (most == 256 && ceil_div(a.m, 256) * ch > sms) return {true, 256, 1};
  const double bytes = (double)ch * kc * Q8_WTILE;
  Q8Plan best{false, most, 1};
  double least = 1e30;
  for (int nt = most;; nt = std::max(16, (int)round_up(nt / 2, 16))) {
    const int64_t row_tiles = ceil_div(a.m, nt);
    for (int s = 1; s <= (nt <= 64 ? 8 : 1) && s <= kc; ++s) {  // a split's sums are stored behind a small ring
      const int64_t turns = ceil_div(row_tiles * ch * s, sms * (nt <= 64 ? 2 : 1));
      const double loop = (double)(turns * ceil_div(kc, s)) * (300 + 0.25 * nt);
      const double stream = bytes / 6200 + (double)(row_tiles - 1) * bytes / 12000;
      const double cost = std::max(loop, stream) + 2000.0 * (double)(turns - 1) + (s > 1 ? 3000.0 : 0.0);
      if (cost < least) {
        least = cost;
        best.nt = nt;
        best.splits = s;
      }
    }
    if (nt <= 32) break;
  }
  return best;
}

template <int OUT>
static bool launch_q8(const Q8Args& a, cudaStream_t st) {
  // Two rows at most (three take as long as a tile of 16), and 16 KB of their codes, which each block loads first: one
  // row of 4096 on 12288 channels takes 12.4 us (the ring 17.2), two 14.5 (17.6); one of 16384 on 4096 16.5 (18.6), of
  // 22016 26.9 (22.7), two of 8192 12.4 (12.8), of 11008 18.6 (14.9).
  const int kc = (int)ceil_div(a.k, Q8_KB);
  if (a.m <= 2 && a.m * kc * Q8_KB <= 16 * 1024) {
    const unsigned grid = (unsigned)ceil_div(a.n, 2 * Q8_VW);
    const size_t sm = (size_t)(a.m * kc * Q8_KB);
    launch_next(a.m == 1 ? q8_vector_kernel<OUT, 1> : q8_vector_kernel<OUT, 2>, dim3(grid), Q8_VW * 32, sm, st, a);
    count_launch();
    return true;
  }
  static OncePerDevice once;
  once([] {
    cudaFuncSetAttribute(q8_split_kernel<OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
    cudaFuncSetAttribute(q8_persistent_kernel<OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 215 * 1024);
  });
  const Q8Plan p = q8_plan(a);
  const int stage = Q8_WTILE + p.nt * Q8_KB;
  CUtensorMap am;
  if (!tma_map_u8(&am, a.a, a.m, a.k, a.lda, Q8_KB, p.nt)) return false;
  Q8Tile t{p.nt, 0, kc, 32, 0};
  while ((int)t.tmem_cols < p.nt) t.tmem_cols *= 2;
  const int ch = (int)ceil_div(a.n, 128);
  const int64_t row_tiles = ceil_div(a.m, p.nt);
  if (p.persistent) {
    t.stages = 4;
    const int64_t tiles = row_tiles * ch;
    q8_persistent_kernel<OUT><<<(unsigned)std::min<int64_t>(tiles, q8_sms()), Q8_PNT, t.stages * stage + 1024, st>>>(
        am, a, t, ch, (int)tiles);
    count_launch();
    return true;
  }
  // the ring and the sums to join: up to 104 KB where two blocks share an SM, else up to 200 KB
  t.join = (int)round_up(ceil_div(p.nt, p.splits), 4);
  const int join = p.splits > 1 ? t.join * p.splits * 128 * 4 : 0;
  t.stages = std::min(12, ((p.nt <= 64 ? 104 : 200) * 1024 - join) / stage);
  const size_t bytes = (size_t)t.stages * stage + join;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = 128;
  cfg.dynamicSmemBytes = bytes + 1024;
  cfg.stream = st;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)p.splits, 1, 1};
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  cfg.gridDim = dim3((unsigned)(ch * p.splits), (unsigned)row_tiles, 1);
  cudaLaunchKernelEx(&cfg, q8_split_kernel<OUT>, am, a, t, p.splits);
  count_launch();
  return true;
}
bool launch_q8_matmul(const Q8Args& a, cudaStream_t st) {
  return a.out_bf16 ? launch_q8<Q8_BF16>(a, st) : a.accumulate ? launch_q8<Q8_ADD>(a, st) : launch_q8<Q8_F32>(a, st);
}

}  // namespace kl
