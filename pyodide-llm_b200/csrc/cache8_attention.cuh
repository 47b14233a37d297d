// cache8_attention.cuh — what the two attention kernels of the paged 8-bit cache share: the call's arguments, a request's
// rows and positions, and the int8 integers as float16.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "common.h"

namespace b200 {
namespace cache8 {

constexpr int UNIT = 16;             // positions of a unit, which lies within one block of the cache
constexpr float RESCALE = 8.0f;      // log2 of how far a weight may rise above 1 before the running maximum moves
// Weights are 2^LIFT where a term is as large as the running maximum, so up to 2^15 before it moves: the upper end of
// float16's range, whose lower end, 2^-24, is then 2^-31 of that term.
constexpr float LIFT = 7.0f;
constexpr float LEAST = 2.019484e-28f;  // 2^-92, see the weights' comment

struct Args {
  void *out;
  const void *q;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *tables, *starts, *lengths;
  int4 *meta;       // [tiles] {first span, spans, request, row tile}; meta[-1]: {the tiles, a wait's error code}
  float2 *part_ml;  // [span + tile][kv head][RT] {M, l}
  float *part;      // [span + tile][kv head][RT][hs]
  int64_t q_stride, out_stride;
  int n, n_seqs, width, blocks, block, nkv, hs, group;
  int min_work, whole_tiles;  // a span's work at least, in units or (whole_tiles) in tiles
  int rows_most;       // a request's rows of a kv head above which it is not cache8_attention.cu's
  float scale;      // log2(e) / sqrt(hs)
};

// request i of the call: its first row, its rows, and its positions (all of them, the new ones included); astray: its
// starts do not ascend within 0..n (the whole call then writes nothing; the rows given here are in bounds all the same)
struct Request {
  int first, fresh, length;
  bool astray;
};
__device__ __forceinline__ Request request_of(const Args &a, int i) {
  const int at = a.starts[i], to = a.starts[i + 1], s0 = min(max(at, 0), a.n), s1 = min(max(to, s0), a.n);
  return {s0, s1 - s0, max(a.lengths[i], 0), s0 != at || s1 != to};
}

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
// two of a word's bytes (already + 128) as float16 integers: 1024 + b is a float16 whose low byte is b
template <uint32_t SEL>
__device__ __forceinline__ uint32_t widen(uint32_t biased) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(biased), "r"(0x64646464u), "n"(SEL));
  const __half2 v = __hsub2(*reinterpret_cast<__half2 *>(&d), __half2half2(__ushort_as_half(0x6480)));  // less 1152
  return *reinterpret_cast<const uint32_t *>(&v);
}

// cache8_attention_tc.cu: the requests of more than ROWS_FEW rows of a kv head. Measured with 8 requests of 2000 positions, 8
// kv heads, here and there: float32 with heads of 64, 16 rows 36 and 37 us, 32 38 and 37, 64 49 and 37, 128 80 and 37;
// with heads of 128, 32 rows 48 and 59, 64 65 and 60, 128 107 and 61; float16 with heads of 128, 32 rows 44 and 42, 64 57
// and 42, 128 92 and 42.
constexpr int ROWS_FEW = 64;
int launch_attention8_prompts(const Args &a, bool half, cudaStream_t stream);
// head sizes that it takes
inline bool prompts_fit(int hs) { return hs <= 128; }

}  // namespace cache8
}  // namespace b200
