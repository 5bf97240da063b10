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

namespace kl {
namespace {

__device__ __forceinline__ bool finite32(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// rint(127 u / top) for u = h * w in 64 bits.  The f32 quotient decides unless
// it is within 1e-4 of a border between two codes (its own error is below
// 3 roundings of 127, 2.3e-5): only then are the 64-bit product and quotient
// taken, so the codes are those of the definition.
__device__ __forceinline__ int q8_code(float h, float w, float p, float inv, double top) {
  const float t = p * inv;
  const float r = rintf(t);
  if (fabsf(fabsf(t - r) - 0.5f) < 1e-4f) return (int)rint((double)h * (double)w * 127.0 / top);
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

// One block per row; the row's h waits in shared memory between the pass that
// finds its sum of squares and maximum and the pass that writes the codes.
template <int NT, class T>
__global__ void __launch_bounds__(NT) norm_q8_kernel(NormQ8Args a) {
  extern __shared__ float nq_h[];
  __shared__ float tmp[NT / 32];
  __shared__ unsigned long long top_s;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const float* r = a.residual ? a.residual + row * a.ldr : nullptr;
  float* ho = a.hidden ? a.hidden + row * a.ldh : nullptr;
  if (threadIdx.x == 0) top_s = 0ull;
  float ss = 0.f, mx = 0.f;
  bool fin = true;
  for (int i = threadIdx.x; i < a.cols; i += NT) {
    float h = to_f(x[i]);
    if (r) h += r[i];
    if (ho) ho[i] = h;
    nq_h[i] = h;
    const float w = a.weight ? (a.one_plus ? 1.f + a.weight[i] : a.weight[i]) : 1.f;
    const float p = h * w;
    fin = fin && finite32(p) && finite32(h);
    ss = fmaf(h, h, ss);
    mx = fmaxf(mx, fabsf(p));
  }
  ss = block_reduce<NT>(ss, tmp, false);
  mx = block_reduce<NT>(fin ? mx : INFINITY, tmp, true);
  // the largest |h w| in 64 bits is among those whose f32 product is largest
  for (int i = threadIdx.x; i < a.cols; i += NT) {
    const float w = a.weight ? (a.one_plus ? 1.f + a.weight[i] : a.weight[i]) : 1.f;
    if (fabsf(nq_h[i] * w) == mx)
      atomicMax(&top_s, (unsigned long long)__double_as_longlong(fabs((double)nq_h[i] * (double)w)));
  }
  __syncthreads();
  const double top = __longlong_as_double((long long)top_s);
  const float rinv = a.norm ? 1.f / sqrtf(ss / (float)a.cols + a.eps) : 1.f;
  const bool good = finite32(mx) && finite32(ss);
  if (threadIdx.x == 0) a.scales[row] = good ? mx * rinv / 127.f : __int_as_float(0x7fffffff);
  const float inv = good && mx > 0.f ? 127.f / mx : 0.f;
  int8_t* co = a.codes + row * a.ldc;
  for (int i = threadIdx.x; i < a.cols; i += NT) {
    const float w = a.weight ? (a.one_plus ? 1.f + a.weight[i] : a.weight[i]) : 1.f;
    co[i] = inv > 0.f ? (int8_t)q8_code(nq_h[i], w, nq_h[i] * w, inv, top) : (int8_t)0;
  }
}

__device__ __forceinline__ void q8_store(const Q8Args& a, int64_t r, int64_t c, int acc) {
  float v = (float)acc * a.a_scale[r] * a.w_scale[c];
  if (a.bias) v += a.bias[c];
  if (a.out_bf16) {
    static_cast<__nv_bfloat16*>(a.out)[r * a.ldo + c] = __float2bfloat16_rn(v);
  } else {
    float* o = static_cast<float*>(a.out) + r * a.ldo + c;
    *o = a.accumulate ? *o + v : v;
  }
}

// One thread per output, four products an instruction.
__global__ void q8_simple_kernel(Q8Args a) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, r = blockIdx.y;
  if (c >= a.n) return;
  const int8_t* x = a.a + r * a.lda;
  const int8_t* w = a.w + c * a.ldw;
  int acc = 0, k = 0;
  for (; k + 4 <= a.k; k += 4)
    acc = __dp4a(*reinterpret_cast<const int*>(x + k), *reinterpret_cast<const int*>(w + k), acc);
  for (; k < a.k; ++k) acc += (int)x[k] * (int)w[k];
  q8_store(a, r, c, acc);
}

__global__ void q8_pack_kernel(const int8_t* src, int64_t ld, int k, int8_t* dst, int64_t ldw) {
  const int64_t r = blockIdx.y;
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c < ldw) dst[r * ldw + c] = c < k ? src[r * ld + c] : (int8_t)0;
}

}  // namespace

void launch_norm_q8(const NormQ8Args& a, int rows, cudaStream_t st) {
  static OncePerDevice once;
  once([] {
    cudaFuncSetAttribute(norm_q8_kernel<256, float>, cudaFuncAttributeMaxDynamicSharedMemorySize, NORM_Q8_MAX_COLS * 4);
    cudaFuncSetAttribute(norm_q8_kernel<256, __nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         NORM_Q8_MAX_COLS * 4);
  });
  const size_t sm = (size_t)a.cols * 4;
  if (a.x_bf16) norm_q8_kernel<256, __nv_bfloat16><<<rows, 256, sm, st>>>(a);
  else norm_q8_kernel<256, float><<<rows, 256, sm, st>>>(a);
  count_launch();
}

void launch_q8_pack(const int8_t* src, int64_t ld, int n, int k, int8_t* dst, int64_t ldw, cudaStream_t st) {
  for (int r = 0; r < n; r += 65535)
    q8_pack_kernel<<<dim3((unsigned)ceil_div(ldw, 256), std::min(65535, n - r)), 256, 0, st>>>(
        src + r * ld, ld, k, dst + r * ldw, ldw), count_launch();
}

void launch_q8_matmul(const Q8Args& a, cudaStream_t st) {
  for (int r = 0; r < a.m; r += 65535) {
    Q8Args b = a;
    b.a += r * a.lda;
    b.a_scale += r;
    b.out = static_cast<char*>(a.out) + r * a.ldo * (a.out_bf16 ? 2 : 4);
    q8_simple_kernel<<<dim3((unsigned)ceil_div(a.n, 128), std::min(65535, a.m - r)), 128, 0, st>>>(b);
    count_launch();
  }
}

}  // namespace kl
