// attend.cu -- attention of a call's new tokens over the paged 4-bit cache
// (kv4.cuh): o = softmax(scale * q . K^T) . V over the keys that a token sees,
// K = ks c + km, V = vs c + vm.  Token i of a sequence (0-based over its whole
// length) sees tokens j <= i, and with a window w only i - w < j.  A token
// that sees nothing gets zeros.
#include "engine.h"
#include "kv4.cuh"

namespace kl {
namespace {

// One warp per (token, query head), a running maximum and sum in 32 bits.
template <int D>
__global__ void attend_simple_kernel(AttendArgs a) {
  constexpr int E = D / 32;  // dims per lane
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = blockIdx.y + blockIdx.z * 65535;
  if (t >= a.seq.num_tokens) return;
  const int b = find_seq(a.seq.cu_q, a.seq.num_seqs, t);
  if (b >= a.seq.num_seqs || head >= a.q_heads) return;
  bool bad = false;
  const int ps = a.cache.page_size, kvh = head / (a.q_heads / a.cache.kv_heads);
  const SeqSpan s = seq_span(a.seq, b, ps, &bad);
  const int index = s.kv_len - s.q_len + (t - s.row);
  const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(a.q.p) + t * a.q.token + head * a.q.head;
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    q[i] = to_f(qp[lane * E + i]) * a.scale;
    o[i] = 0.f;
  }
  const int first = a.window > 0 ? max(0, index - a.window + 1) : 0;
  for (int j = first; j <= index; ++j) {
    const int64_t page = a.seq.table[b * a.seq.table_ld + j / ps];
    if (page < 0 || page >= a.cache.num_pages) {
      bad = true;
      continue;
    }
    const int off = j % ps, tok = off & 15;
    const unsigned char* tile = kv4_tile(a.cache, kv4_tile_bytes(D), page, kvh, off >> 4);
    const uint2 pr = *reinterpret_cast<const uint2*>(tile + 2 * kv4_codes(D) + tok * 8);
    const int w = lane * E / 8;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(tile + kv4_k_off<D>(tok, w));
    const uint32_t vw = *reinterpret_cast<const uint32_t*>(tile + kv4_codes(D) + kv4_v_off<D>(tok, w));
    const float ks = __uint_as_float(pr.x << 16), km = __uint_as_float(pr.x & 0xffff0000u);
    const float vs = __uint_as_float(pr.y << 16), vm = __uint_as_float(pr.y & 0xffff0000u);
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = (lane * E + i) & 7;
      x = fmaf(q[i], fmaf((float)((kw >> (4 * kv4_nibble(e))) & 15u), ks, km), x);
    }
    x = warp_sum_f(x);
    const float mn = fmaxf(m, x), ref = mn == -INFINITY ? 0.f : mn;
    const float keep = expf(m - ref), p = expf(x - ref);
    m = mn;
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = (lane * E + i) & 7;
      o[i] = fmaf(p, fmaf((float)((vw >> (4 * kv4_nibble(e))) & 15u), vs, vm), o[i] * keep);
    }
  }
  if (bad && lane == 0) atomicOr(a.err, DERR_BOUNDS);
  __nv_bfloat16* op = static_cast<__nv_bfloat16*>(a.out.p) + t * a.out.token + head * a.out.head;
#pragma unroll
  for (int i = 0; i < E; ++i) op[lane * E + i] = __float2bfloat16_rn(l == 0.f ? 0.f : o[i] / l);
}

}  // namespace

size_t attend_workspace(const AttendShape&) { return 0; }

void launch_attend(const AttendArgs& a, const AttendShape& s, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.q_heads, 4), (unsigned)std::min(a.seq.num_tokens, 65535),
                  (unsigned)ceil_div(a.seq.num_tokens, 65535));
  if (s.D == 128) attend_simple_kernel<128><<<grid, 128, 0, st>>>(a);
  else attend_simple_kernel<64><<<grid, 128, 0, st>>>(a);
  count_launch();
}

}  // namespace kl
