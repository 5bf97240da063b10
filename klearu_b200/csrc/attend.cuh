// attend.cuh -- device code shared by the attention kernels.
#pragma once

#include "kv4.cuh"

namespace kl {

// attend_tc.cu; with more than one chunk of the keys the join is the caller's
void launch_attend_tc(const AttendArgs& a, const AttendShape& s, int chunks, cudaStream_t st);

// 2^x by the special function unit; results below 2^-126 are zero
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// The first token that token pos sees (0 where pos is a row in front of its sequence); a window may be as large as a
// number gets, a position as small, so the difference is not taken where it would be negative.
__device__ __forceinline__ int window_from(int window, int pos) { return window > 0 && pos >= window ? pos - window + 1 : 0; }

// The workspace: (reference, sum) of [chunk][token][query head], then their rows of D.
__device__ __forceinline__ float* join_rows(const AttendArgs& a, int chunks) {
  const int64_t n = (int64_t)chunks * a.seq.num_tokens * a.q_heads * 2;
  return a.scratch + ((n + 3) & ~(int64_t)3);
}

__device__ __forceinline__ void attend_store4(const HeadRows& out, int64_t tok, int head, int d, const float* v,
                                              float f) {
  __nv_bfloat16* p = static_cast<__nv_bfloat16*>(out.p) + tok * out.token + head * out.head + d;
  const uint32_t x = pack_bf16(v[0] * f, v[1] * f), y = pack_bf16(v[2] * f, v[3] * f);
  if (out.vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(x, y);
  } else {
    unsigned short* s = reinterpret_cast<unsigned short*>(p);
    s[0] = (unsigned short)(x & 0xffffu);
    s[1] = (unsigned short)(x >> 16);
    s[2] = (unsigned short)(y & 0xffffu);
    s[3] = (unsigned short)(y >> 16);
  }
}

}  // namespace kl
