// cache8.cu — the paged 8-bit key/value cache: b200k_block_tables (which block of the pool holds which positions of
// which request), b200k_cache8_store (keys and values into their blocks) and b200k_cache8_load (out of them again).
//
// A pool of `blocks` blocks, each of `block` positions: values int8 [blocks][kv head][block][head size], one float32
// scale per (block, kv head); keys and values have a pool each. A (block, head) is contiguous, so the attention reads
// whole rows of a head and one scale serves a run of positions. Position p of a request sits in slot
// tables[request][p / block] * block + p % block.
#include <cuda_fp16.h>

#include <cstdint>
#include <string>

#include "cache8.h"
#include "common.h"

namespace b200 {
namespace {

// x / by for 0 <= x < 2^31 and by from 16 to 256, inverse = ceil(2^32 / by): the product is never below the quotient, and
// one above at most
__host__ __device__ inline uint32_t inverse_of(int by) { return 0xffffffffu / (uint32_t)by + 1; }
__device__ __forceinline__ int over(int x, int by, uint32_t inverse) {
  const int q = (int)__umulhi((uint32_t)x, inverse);
  return (uint32_t)q * (uint32_t)by > (uint32_t)x ? q - 1 : q;
}

// ------------------------------------------------------------------------------------------------ block tables
//
// L' = max(0, L + news) positions a request: its blocks go from ceil(L / block) to ceil(L' / block), new ones taken
// from the head of the ring of free ids in the requests' order, blocks left behind put at its tail. Bound by latency:
// a step of 64 requests moves 2 KB. So one launch does it all: one block, or one cluster of eight where there is more
// to write, and every block of the cluster adds up all requests by itself (8 bytes each, from L2) instead of waiting
// for partial sums. Takes read the ring's live part and gives write behind it, takes write table entries that no
// token's slot is read from (a token of a new block finds its id in the ring), so only lengths and state, which may
// be updated in place, have to wait until every block has read them: the one cluster barrier.
// Steps of more than ROWS_APART rows have them written by a second launch, on all SMs: 1000 requests of 64 tokens each take
// 14 us so and 20 with the cluster writing them, 64 of 512 8 and 9, 64 of 64 (the bound's other side) 8 by one block.
// Measured: 64 requests of a token each 5.8 us; 1000 that add 250 to 500 tokens each (358,000 rows) 15.8 us, of which the
// sums over 1000 requests, by every block, are most. A launch by itself is 2 to 3 us.

constexpr int TT = 512;  // threads, and the requests of one tile of the running sums
constexpr int ROWS_APART = 4096;  // a step's rows that the first launch writes at most

struct Need {
  int64_t tokens, take, give;
};

// what request i asks for; `bad` collects B200K_TABLES_* of requests that cannot have it
__device__ __forceinline__ Need need_of(int64_t length, int64_t add, int64_t most, int block, uint32_t inverse, int &bad,
                                        int64_t &after) {
  if (length < 0 || length > most) {
    bad |= 1 << B200K_TABLES_INPUT;
    after = length;
    return {0, 0, 0};
  }
  after = length + add;
  if (after < 0) after = 0;
  if (after > most) {
    bad |= 1 << B200K_TABLES_WIDTH;
    return {0, 0, 0};
  }
  const int before_b = over((int)length + block - 1, block, inverse), after_b = over((int)after + block - 1, block, inverse);
  return {add > 0 ? add : 0, after_b > before_b ? after_b - before_b : 0, before_b > after_b ? before_b - after_b : 0};
}

__device__ __forceinline__ int64_t warp_scan(int64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// the request (an index into the tile's exclusive sums, sums[count] the total) whose part holds item t
__device__ __forceinline__ int find(const int *sums, int count, int t) {
  int lo = 0, hi = count;  // sums[lo] <= t < sums[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct TablesArgs {
  int32_t *tables, *ring, *state_out, *lengths_out, *starts, *slots, *seq, *pos;
  const int32_t *state, *lengths, *news;
  int n_seqs, width, blocks, block, n;
  int apart;  // the tokens' rows are written by a kernel of their own
};

__global__ void __launch_bounds__(TT) block_tables_kernel(TablesArgs a) {
  pdl_begin();
  __shared__ int64_t part[3][TT / 32];
  __shared__ int sums[3][TT + 1], len_s[TT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int64_t most = (int64_t)a.width * a.block;
  const int head = a.state[0], count = a.state[1];
  const uint32_t inverse = inverse_of(a.block);
  auto over_block = [&](int x) { return over(x, a.block, inverse); };

  // this thread's request of a tile, what it needs, and the sums of that before it and over the tile
  int length = 0, bad = 0;
  int64_t after = 0, run[3], all[3];
  Need need = {0, 0, 0};
  auto tile_of = [&](int base) {
    const int i = base + tid;
    need = {0, 0, 0};
    length = 0;
    if (i < a.n_seqs) {
      length = a.lengths[i];
      need = need_of(length, a.news[i], most, a.block, inverse, bad, after);
    }
    const int64_t own[3] = {need.tokens, need.take, need.give};
#pragma unroll
    for (int j = 0; j < 3; j++) run[j] = warp_scan(own[j]);
    __syncthreads();  // (the tile before has been read)
    if (lane == 31) part[0][warp] = run[0], part[1][warp] = run[1], part[2][warp] = run[2];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 3; j++) {
      int64_t before = 0;
      all[j] = 0;
#pragma unroll
      for (int w = 0; w < TT / 32; w++) {
        if (w < warp) before += part[j][w];
        all[j] += part[j][w];
      }
      run[j] += before - own[j];
    }
  };

  // what everything comes to: all is granted, or nothing is
  int64_t sum[3] = {0, 0, 0};
  if (a.n_seqs <= TT) {
    tile_of(0);
#pragma unroll
    for (int j = 0; j < 3; j++) sum[j] = all[j];
  } else {
#pragma unroll 2
    for (int i = tid; i < a.n_seqs; i += TT) {
      const Need one = need_of(a.lengths[i], a.news[i], most, a.block, inverse, bad, after);
      sum[0] += one.tokens, sum[1] += one.take, sum[2] += one.give;
    }
#pragma unroll
    for (int j = 0; j < 3; j++) {
#pragma unroll
      for (int d = 16; d; d >>= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], d);
      if (lane == 0) part[j][warp] = sum[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 3; j++) {
      sum[j] = 0;
#pragma unroll
      for (int w = 0; w < TT / 32; w++) sum[j] += part[j][w];
    }
  }
  bad = __syncthreads_or(bad & 1 << B200K_TABLES_INPUT) ? 1 << B200K_TABLES_INPUT
        : __syncthreads_or(bad & 1 << B200K_TABLES_WIDTH) ? 1 << B200K_TABLES_WIDTH : 0;
  if (head < 0 || head >= a.blocks || count < 0 || count > a.blocks || count + sum[2] > a.blocks)
    bad = 1 << B200K_TABLES_INPUT;
  if (sum[0] > a.n) bad |= 1 << B200K_TABLES_TOKENS;
  if (sum[1] > count) bad |= 1 << B200K_TABLES_BLOCKS;
  const bool granted = bad == 0;
  const int total = granted ? (int)sum[0] : 0;
  auto in_ring = [&](int u) {  // the ring's place u after its head, u below 2^31 - blocks
    const int at = head + u;
    return at >= a.blocks ? at - a.blocks : at;
  };

  const int stride = (int)ranks * TT, first = (int)rank * TT + tid;
  int carry[3] = {0, 0, 0};
  if (granted) {
    for (int base = 0; base < a.n_seqs; base += TT) {
      const int tile = min(TT, a.n_seqs - base);
      if (a.n_seqs > TT) tile_of(base);
      len_s[tid] = length;
#pragma unroll
      for (int j = 0; j < 3; j++) {
        sums[j][tid] = (int)(carry[j] + run[j]);
        if (tid == 0) sums[j][TT] = (int)(carry[j] + all[j]);
      }
      __syncthreads();
      if (tid < tile && rank == 0) a.starts[base + tid] = sums[0][tid];
      // the tokens of this tile of requests, their slots from the table or, in blocks taken now, from the ring; a few of
      // them at a time, so that their lookups overlap
      constexpr int AT_ONCE = 4;
      for (int t0 = a.apart ? sums[0][TT] : carry[0] + first; t0 < sums[0][TT]; t0 += AT_ONCE * stride) {
        int s[AT_ONCE], p[AT_ONCE], id[AT_ONCE], b[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; k++) s[k] = find(sums[0], tile, min(t0 + k * stride, sums[0][TT] - 1));
#pragma unroll
        for (int k = 0; k < AT_ONCE; k++) {
          p[k] = len_s[s[k]] + (min(t0 + k * stride, sums[0][TT] - 1) - sums[0][s[k]]);
          b[k] = over_block(p[k]);
          const int held = over_block(len_s[s[k]] + a.block - 1);
          id[k] = b[k] < held ? a.tables[(int64_t)(base + s[k]) * a.width + b[k]] : a.ring[in_ring(sums[1][s[k]] + (b[k] - held))];
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; k++) {
          const int t = t0 + k * stride;
          if (t >= sums[0][TT]) break;
          a.slots[t] = id[k] >= 0 && id[k] < a.blocks ? id[k] * a.block + (p[k] - b[k] * a.block) : -1;
          if (a.seq) a.seq[t] = base + s[k];
          if (a.pos) a.pos[t] = p[k];
        }
      }
      for (int u = carry[1] + first; u < sums[1][TT]; u += stride) {
        const int s = find(sums[1], tile, u), held = over_block(len_s[s] + a.block - 1);
        a.tables[(int64_t)(base + s) * a.width + held + (u - sums[1][s])] = a.ring[in_ring(u)];
      }
      for (int u = carry[2] + first; u < sums[2][TT]; u += stride) {
        // request s keeps its first held - (its gives) blocks
        const int s = find(sums[2], tile, u), held = over_block(len_s[s] + a.block - 1), gives = sums[2][s + 1] - sums[2][s];
        a.ring[((int64_t)head + count + u) % a.blocks] =
            a.tables[(int64_t)(base + s) * a.width + held - gives + (u - sums[2][s])];
      }
#pragma unroll
      for (int j = 0; j < 3; j++) carry[j] = sums[j][TT];
    }
  } else if (rank == 0) {
    for (int i = tid; i < a.n_seqs; i += TT) a.starts[i] = 0;
  }
  if (rank == 0 && tid == 0) a.starts[a.n_seqs] = total;
  // rows of the step's buffers behind its tokens
  for (int t = a.apart ? a.n : total + first; t < a.n; t += stride) {
    a.slots[t] = -1;
    if (a.seq) a.seq[t] = -1;
    if (a.pos) a.pos[t] = -1;
  }
  // lengths and state may be updated in place: not before every block has read them
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
  for (int i = first; i < a.n_seqs; i += stride) {
    if (a.n_seqs > TT || ranks > 1) {
      length = a.lengths[i];
      int none = 0;
      need_of(length, a.news[i], most, a.block, inverse, none, after);
    }
    a.lengths_out[i] = granted ? (int)after : length;
  }
  if (rank == 0 && tid == 0) {
    int status = 0;
    if (bad & (1 << B200K_TABLES_BLOCKS)) status = B200K_TABLES_BLOCKS;
    if (bad & (1 << B200K_TABLES_TOKENS)) status = B200K_TABLES_TOKENS;
    if (bad & (1 << B200K_TABLES_WIDTH)) status = B200K_TABLES_WIDTH;
    if (bad & (1 << B200K_TABLES_INPUT)) status = B200K_TABLES_INPUT;
    a.state_out[0] = granted ? (int)((head + sum[1]) % a.blocks) : head;
    a.state_out[1] = granted ? (int)(count - sum[1] + sum[2]) : count;
    a.state_out[2] = status;
    a.state_out[3] = total;
  }
}

// The rows of a step of many tokens, from what block_tables_kernel has written: a warp takes CHUNK of them side by side,
// finds the first one's request in the running sums, the last one's, and each token's between them.
constexpr int RT_THREADS = 256, CHUNK = 128;
__global__ void __launch_bounds__(RT_THREADS) block_rows_kernel(TablesArgs a) {
  pdl_begin();
  const int lane = threadIdx.x & 31, t0 = (blockIdx.x * (RT_THREADS / 32) + (threadIdx.x >> 5)) * CHUNK;
  if (t0 >= a.n) return;
  const int total = a.starts[a.n_seqs], last = min(t0 + CHUNK, total) - 1;
  const uint32_t inverse = inverse_of(a.block);
  // the request whose rows hold t, of those from lo to hi (none below hi starts behind t)
  auto request_of = [&](int t, int lo, int hi) {
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.starts[mid] <= t) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  int low = 0, high = 1;
  if (t0 < total) {
    low = request_of(t0, 0, a.n_seqs);
    high = last < a.starts[low + 1] ? low + 1 : request_of(last, low, a.n_seqs) + 1;
  }
#pragma unroll
  for (int k = 0; k < CHUNK / 32; k++) {
    const int t = t0 + 32 * k + lane;
    if (t >= a.n) return;
    int slot = -1, s = -1, p = -1;
    if (t < total) {
      s = request_of(t, low, high);
      p = a.lengths_out[s] - (a.starts[s + 1] - t);
      const int b = over(p, a.block, inverse), id = a.tables[(int64_t)s * a.width + b];
      if (id >= 0 && id < a.blocks) slot = id * a.block + (p - b * a.block);
    }
    a.slots[t] = slot;
    if (a.seq) a.seq[t] = s;
    if (a.pos) a.pos[t] = p;
  }
}

// ------------------------------------------------------------------------------------------------------- store
//
// A (block, head)'s scale is s = max |x| / 127 in float32 over all that it holds, and every value is the integer
// nearest to x / s, half to even, of the real quotient: a float32 guess, and where its remainder comes near half a step,
// the exact one. A token that raises the scale of a block with earlier tokens in it has their integers q brought to the
// new step, nearest(q s_old / s): one scale a block costs that, and only blocks that a request still fills pay it.
//
// Tokens of a block stand together in the call (a request's positions do), so the block's work belongs to the place
// where its run of tokens begins: no two teams touch one (block, head), and no atomics. A team is a thread block, or a
// warp where the call has few tokens; it keeps the values that fit its registers between finding the largest and
// rounding (the rest it reads again, from L1).
// Measured with the load that follows, 8 heads of 128: 64 single tokens in float32 7.5 us (a thread block a token 9.5),
// 4700 tokens of 64 prompts in float16 35 us where the rows are in L2, else 42, of which the load is 12 (a warp a run: 54
// together). Bound by instructions
// and their latency: a run's slots, scale and largest value come one after the other.

constexpr int ST = 128;  // threads of a block
constexpr int KEEP = 4;  // 16-byte vectors of new values that a thread keeps in registers between its two passes

__device__ __forceinline__ void values_of(const uint4 &u, float (&x)[4]) {
  x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void values_of(const uint4 &u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}

// What kernels before this one in the stream may write while this one is already there (its wait is at its beginning), so
// no loads for memory that stays as it is; volatile, so none comes before that wait, and not held back by the stores
// between them, which go elsewhere.
__device__ __forceinline__ uint4 vector_at(const void *p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ int slot_at(const int32_t *p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

// the integer nearest to q a / b, half to even, in 64 bits: q a is exact there (q an integer of 8 bits, or 1 and a a
// float), and so far from a half that is not one that the quotient's rounding cannot reach it. At most 127 in size: a
// scale of a few of float32's smallest steps may be a third below the largest value's 127th part (and has no inverse, so
// all its values come here).
__device__ __noinline__ int exactly(double qa, double b) { return (int)fmin(fmax(rint(__ddiv_rn(qa, b)), -127.0), 127.0); }

// the largest |x|: NaN above infinity above every number
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
template <int VW>
__device__ __forceinline__ float largest(float top, const uint4 &u) {
  float x[VW];
  values_of(u, x);
#pragma unroll
  for (int i = 0; i < VW; i++) top = max_nan(top, fabsf(x[i]));
  return top;
}

// four integers as bytes: t = 1.5 2^23 + (x / s rounded) has the integer in its low bits, and x - q s is exact (a multiple
// of s's last place, and no larger than about s), so it tells whether the integer is the nearest one, or has a rival
__device__ __forceinline__ uint32_t four_bytes(const float *x, float s, float inv) {
  float off = 0.0f;
  uint32_t t[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float z = __fmaf_rn(x[j], inv, 12582912.0f);
    t[j] = __float_as_uint(z);
    off = fmaxf(off, fabsf(__fmaf_rn(-(z - 12582912.0f), s, x[j])));
  }
  if (off + off >= s) {
#pragma unroll 1
    for (int j = 0; j < 4; j++) t[j] = (uint32_t)exactly(x[j], s);
  }
  return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}
// four earlier integers from scale a to scale b, ratio about a / b (q a is rounded here: by 2^-24 of 127 b at most; where b
// is a few of float32's smallest steps the margin rounds to b itself, and a tie has to be let through)
__device__ __forceinline__ uint32_t four_moved(uint32_t q4, float a, float b, float ratio) {
  float off = 0.0f;
  uint32_t t[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float q = (float)(int8_t)(q4 >> (8 * j)), z = __fmaf_rn(q, ratio, 12582912.0f);
    t[j] = __float_as_uint(z);
    off = fmaxf(off, fabsf(__fmaf_rn(-(z - 12582912.0f), b, __fmul_rn(q, a))));
  }
  if (off + off >= b * 0.99997f) {
#pragma unroll 1
    for (int j = 0; j < 4; j++) t[j] = (uint32_t)exactly((double)(int8_t)(q4 >> (8 * j)) * a, b);
  }
  return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}

struct StoreArgs {
  int8_t *cache[2];
  float *scales[2];
  const void *x[2];
  int64_t stride[2];
  const int32_t *slots;
  int n, blocks, block, nkv, hs, per;
};

// A team (TEAM threads: a block, or a warp of one) a head, its keys or its values, for the runs that begin among `per`
// tokens.
template <bool HALF, int TEAM>
__global__ void __launch_bounds__(ST, 8) cache8_store_kernel(StoreArgs a) {
  pdl_begin();
  constexpr int VW = HALF ? 8 : 4;  // values of a 16-byte vector
  __shared__ float top_s[2][ST / 32];
  const int lane = threadIdx.x & 31, tid = threadIdx.x % TEAM;
  const int unit = TEAM == ST ? blockIdx.y : blockIdx.y * (ST / TEAM) + threadIdx.x / TEAM;
  if (unit >= 2 * a.nkv) return;
  const bool second = unit >= a.nkv;
  const int h = second ? unit - a.nkv : unit;
  int8_t *cache = second ? a.cache[1] : a.cache[0];
  float *scales = second ? a.scales[1] : a.scales[0];
  const int64_t step = (second ? a.stride[1] : a.stride[0]) * (HALF ? 2 : 4);
  const int i0 = blockIdx.x * a.per, i1 = min(a.n, i0 + a.per);
  // a row by vpr threads, `rows` rows at a time (a row of more vectors than a warp has lanes: in two parts)
  const int vectors = a.hs / VW, parts = vectors > TEAM ? 2 : 1, vpr = vectors / parts, rows = TEAM / vpr;
  const int row = tid / vpr, col = (tid - row * vpr) * VW;
  const char *x = reinterpret_cast<const char *>(second ? a.x[1] : a.x[0]) + (int64_t)i0 * step +
                  ((int64_t)h * a.hs + col) * (HALF ? 2 : 4);
  // a single token's vector, on its way before its slot is known
  uint4 first = make_uint4(0, 0, 0, 0);
  if (TEAM < ST && row == 0) first = vector_at(x);
  const uint32_t inverse = inverse_of(a.block);
  // the block of token i, or -1 (a lane a token, every warp by itself)
  auto page_of = [&](int i) {
    const int slot = i >= 0 && i < a.n ? slot_at(a.slots + i) : -1;
    const int page = slot < 0 ? -1 : over(slot, a.block, inverse);
    return page < a.blocks ? page : -1;
  };
  const int mine = page_of(i0 + lane), next = page_of(i0 + lane + 1);
  int before = __shfl_up_sync(0xffffffffu, mine, 1);
  if (lane == 0) before = page_of(i0 - 1);
  uint32_t begins = __ballot_sync(0xffffffffu, i0 + lane < i1 && mine >= 0 && mine != before);
  const uint32_t ends = __ballot_sync(0xffffffffu, mine != next);  // the last token of its block's run
  int turn = 0;
  for (; begins; begins &= begins - 1) {
    const int k = __ffs(begins) - 1, i = i0 + k, page = __shfl_sync(0xffffffffu, mine, k);
    const int slot = slot_at(a.slots + i), held = slot - page * a.block;  // held: earlier tokens in the block
    float *scale = scales + (int64_t)page * a.nkv + h;
    const float s_old = held ? *scale : 0.0f;
    const uint32_t end = ends >> k;
    int m = end ? __ffs(end) : 32 - k;  // the run of tokens of this block, at least so far as these 32 go
    while (!end) {
      const uint32_t other = __ballot_sync(0xffffffffu, page_of(i + m + lane) != page);
      if (other) {
        m += __ffs(other) - 1;
        break;
      }
      m += 32;
    }
    // this thread's vectors: of rows row, row + rows, ..., a row's parts one after the other
    const int mine_of = row < rows ? (m * parts - row + rows - 1) / rows : 0;
    const char *src = x + k * step;
    auto vector = [&](int u) {
      const int r = row + u * rows, t = parts == 2 ? r >> 1 : r;
      return vector_at(src + t * step + (parts == 2 ? (r & 1) * vpr * 16 : 0));
    };
    uint4 kept[KEEP];
    float top = 0.0f;
#pragma unroll
    for (int u = 0; u < KEEP; u++)
      if (u < mine_of) kept[u] = TEAM < ST && u == 0 && row == 0 && k == 0 ? first : vector(u);
#pragma unroll
    for (int u = 0; u < KEEP; u++)
      if (u < mine_of) top = largest<VW>(top, kept[u]);
#pragma unroll 4
    for (int u = KEEP; u < mine_of; u++) top = largest<VW>(top, vector(u));
#pragma unroll
    for (int d = 16; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (TEAM == ST) {
      // (by turns: a warp may be a run ahead of another that still reads)
      if (lane == 0) top_s[turn][threadIdx.x >> 5] = top;
      __syncthreads();  // (and this run's scale has been read)
#pragma unroll
      for (int w = 0; w < ST / 32; w++) top = max_nan(top, top_s[turn][w]);
      turn ^= 1;
    }
    // a value that is no finite number, now or among the earlier ones, makes the block's scale NaN: its values read
    // as NaN until the block is begun again
    float s = top < INFINITY ? __fdiv_rn(top, 127.0f) : __uint_as_float(0x7fffffffu);
    if (!(s_old <= s)) s = s != s ? s : s_old;
    const float inv = s > 1e-37f ? __fdiv_rn(1.0f, s) : 0.0f;
    int8_t *dst = cache + ((int64_t)page * a.nkv + h) * a.block * a.hs;
    if (TEAM < ST) __syncwarp();  // (every lane has read the scale)
    if (tid == 0) *scale = s;
    if (s > s_old && s_old > 0) {
      // the earlier tokens' integers to the new step
      const float ratio = __fdiv_rn(s_old, s);
      uint4 *q16 = reinterpret_cast<uint4 *>(dst);
#pragma unroll 2
      for (int w = tid; w < held * a.hs / 16; w += TEAM) {
        const uint4 q = q16[w];
        q16[w] = make_uint4(four_moved(q.x, s_old, s, ratio), four_moved(q.y, s_old, s, ratio),
                            four_moved(q.z, s_old, s, ratio), four_moved(q.w, s_old, s, ratio));
      }
    }
    // s 0: the block holds zeros (or values under half a step of the smallest float); s NaN: it held none. A scale so
    // small that its inverse is no float: exactly() throughout (inv is 0 then, every guess 0)
    const bool some = s > 0;
    const int32_t *slots = a.slots + i;
    const int base = page * a.block;
    dst += col;
    auto one = [&](int u, const uint4 &v) {
      const int r = row + u * rows, t = parts == 2 ? r >> 1 : r;
      float y[VW];
      values_of(v, y);
      int8_t *q = dst + (slot_at(slots + t) - base) * a.hs + (parts == 2 ? (r & 1) * vpr * VW : 0);
      if (HALF)
        *reinterpret_cast<uint2 *>(q) = some ? make_uint2(four_bytes(y, s, inv), four_bytes(y + VW - 4, s, inv)) : make_uint2(0, 0);
      else *reinterpret_cast<uint32_t *>(q) = some ? four_bytes(y, s, inv) : 0;
    };
#pragma unroll
    for (int u = 0; u < KEEP; u++)
      if (u < mine_of) one(u, kept[u]);
#pragma unroll 2
    for (int u = KEEP; u < mine_of; u++) one(u, vector(u));
  }
}

// -------------------------------------------------------------------------------------------------------- load
//
// q s, rounded once to the output's type. Bound by its writes (4 or 2 bytes a value for the 1 read): a thread keeps
// its columns for several tokens and writes 16 bytes a token. Bytes become numbers by a permute under 2^23's exponent and
// a subtraction, four at a time. 4700 tokens of 8 heads of 128 in float16: 12 us for 29 MB.

constexpr int LT = 256;      // threads
constexpr int L_TOKENS = 4;  // tokens of a thread

struct LoadArgs {
  void *out[2];
  const int8_t *cache[2];
  const float *scales[2];
  int64_t stride[2];
  const int32_t *slots;
  int n, blocks, block, nkv, hs;
};

template <bool HALF>
__global__ void __launch_bounds__(LT) cache8_load_kernel(LoadArgs a) {
  pdl_begin();
  constexpr int VW = HALF ? 8 : 4;
  const bool second = blockIdx.z;  // keys, then values
  const int8_t *cache = second ? a.cache[1] : a.cache[0];
  const float *scales = second ? a.scales[1] : a.scales[0];
  char *out = reinterpret_cast<char *>(second ? a.out[1] : a.out[0]);
  const int64_t stride = second ? a.stride[1] : a.stride[0];
  const int v = blockIdx.y * LT + threadIdx.x, vpr = a.nkv * a.hs / VW;
  if (v >= vpr) return;
  const int h = v * VW / a.hs, col = v * VW - h * a.hs;
  const int64_t slots_in = (int64_t)a.blocks * a.block;
  const uint32_t inverse = inverse_of(a.block);
  const int i0 = blockIdx.x * L_TOKENS;
  int slot[L_TOKENS];
  uint2 q[L_TOKENS];
  float s[L_TOKENS];
#pragma unroll
  for (int t = 0; t < L_TOKENS; t++) {
    slot[t] = i0 + t < a.n ? a.slots[i0 + t] : -1;
    if (slot[t] >= slots_in) slot[t] = -1;
  }
#pragma unroll
  for (int t = 0; t < L_TOKENS; t++) {
    if (slot[t] < 0) continue;
    const int page = over(slot[t], a.block, inverse), at = slot[t] - page * a.block;
    const int64_t ph = (int64_t)page * a.nkv + h;
    const int8_t *src = cache + (ph * a.block + at) * a.hs + col;
    if (HALF) q[t] = *reinterpret_cast<const uint2 *>(src);
    else q[t].x = *reinterpret_cast<const uint32_t *>(src);
    s[t] = scales[ph];
  }
#pragma unroll
  for (int t = 0; t < L_TOKENS; t++) {
    if (slot[t] < 0) continue;
    // a byte less its bias is a float's low bits: 2^23 + 128 + q (converting takes the slow pipe)
    float x[VW];
#pragma unroll
    for (int j = 0; j < VW; j++) {
      const uint32_t w = (j < 4 ? q[t].x : q[t].y) ^ 0x80808080u;
      x[j] = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + (j & 3))) - 8388736.0f, s[t]);
    }
    char *dst = out + ((int64_t)(i0 + t) * stride + (int64_t)v * VW) * (HALF ? 2 : 4);
    if (HALF) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const __half2 p = __floats2half2_rn(x[2 * j % VW], x[(2 * j + 1) % VW]);
        w[j] = *reinterpret_cast<const uint32_t *>(&p);
      }
      *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
}

bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

int check_cache8(const char *what, const void *kc, const void *ks, const void *vc, const void *vs, int blocks,
                 int block, int nkv, int hs) {
  const std::string name(what);
  if (!kc || !ks || !vc || !vs) return fail(B200FWD_EINVAL, name + ": null cache");
  if (block < 16 || block > 256 || block % 16)
    return fail(B200FWD_EINVAL, name + ": a block is a multiple of 16 positions, at most 256");
  if (hs < 16 || hs > 256 || hs % 16)
    return fail(B200FWD_EINVAL, name + ": the head size is a multiple of 16, at most 256");
  if (nkv < 1 || nkv > 1024) return fail(B200FWD_EINVAL, name + ": 1 to 1024 kv heads");
  if (blocks < 1 || (int64_t)blocks * block > INT32_MAX)
    return fail(B200FWD_EINVAL, name + ": 1 block at least, and slots that an int32 holds");
  if (!aligned(kc, 16) || !aligned(vc, 16)) return fail(B200FWD_EINVAL, name + ": the cache must be 16-byte aligned");
  return 0;
}

namespace {

// rows of n vectors that the kernels read and write 16 bytes at a time
int check_rows(const char *what, const void *x, int64_t stride, int64_t row, bool half) {
  const std::string name(what);
  if (!x) return fail(B200FWD_EINVAL, name + ": null rows");
  if (stride < row) return fail(B200FWD_EINVAL, name + ": a stride below the row's length");
  if (!aligned(x, 16) || stride % (half ? 8 : 4))
    return fail(B200FWD_EINVAL, name + ": rows must start on 16 bytes");
  return 0;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200k_block_tables(int32_t *tables, int32_t *ring, int32_t *state_out, int32_t *lengths_out,
                                  int32_t *starts, int32_t *slots, int32_t *seq, int32_t *pos, const int32_t *state,
                                  const int32_t *lengths, const int32_t *news, int32_t n_seqs, int32_t table_width,
                                  int32_t blocks, int32_t block, int32_t n, b200fwd_stream stream) {
  try {
    if (!tables || !ring || !state_out || !lengths_out || !starts || !state || !lengths || !news || (n > 0 && !slots))
      return fail(B200FWD_EINVAL, "block_tables: null pointer");
    if (n_seqs < 1 || n_seqs > 1 << 20 || n < 0 || n > 1 << 30)
      return fail(B200FWD_EINVAL, "block_tables: 1 to 2^20 requests, 0 to 2^30 tokens");
    if (block < 16 || block > 256 || block % 16)
      return fail(B200FWD_EINVAL, "block_tables: a block is a multiple of 16 positions, at most 256");
    if (blocks < 1 || (int64_t)blocks * block > INT32_MAX || table_width < 1 ||
        (int64_t)table_width * block > INT32_MAX / 2)
      return fail(B200FWD_EINVAL, "block_tables: 1 block at least, and positions and slots that an int32 holds");
    TablesArgs a = {tables, ring, state_out, lengths_out, starts, slots, seq, pos, state, lengths, news,
                    n_seqs, table_width, blocks, block, n, n > ROWS_APART};
    // One block up to 4096 tokens and 2 tiles of requests, else a cluster of eight. Measured, one and eight: 64 requests of a
    // token each 5.4 and 6.2 us, 64 of 64 tokens 8.0 and 6.3, 1000 of one 12.7 and 13.1, 1025 of three 15.0 and 14.9, 1000
    // of 64 16.4 and 14.3.
    const unsigned ranks = n <= 4096 && n_seqs <= 2 * TT ? 1 : 8;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks);
    cfg.blockDim = dim3(TT);
    cfg.stream = as_stream(stream);
    cfg.attrs = attr;
    cfg.numAttrs = pdl_on() ? 2 : 1;
    (void)cudaLaunchKernelEx(&cfg, block_tables_kernel, a);
    B200_LAUNCHED("block_tables");
    if (a.apart) {
      const int per_block = RT_THREADS / 32 * CHUNK;
      launch(block_rows_kernel, dim3((n + per_block - 1) / per_block), dim3(RT_THREADS), 0, as_stream(stream), a);
      B200_LAUNCHED("block_rows");
    }
    return 0;
  } catch (...) {
    return fail(B200FWD_EINVAL, "block_tables: exception");
  }
}

extern "C" int b200k_cache8_store(int8_t *kc, float *ks, int8_t *vc, float *vs, const void *k, const void *v,
                                  const int32_t *slots, int32_t n, int64_t k_stride, int64_t v_stride, int32_t blocks,
                                  int32_t block, int32_t nkv, int32_t hs, int32_t half, b200fwd_stream stream) {
  try {
    int rc = check_cache8("cache8_store", kc, ks, vc, vs, blocks, block, nkv, hs);
    if (rc) return rc;
    if (n < 0 || n > 1 << 30) return fail(B200FWD_EINVAL, "cache8_store: 0 to 2^30 tokens");
    if (n == 0) return 0;
    if (!slots) return fail(B200FWD_EINVAL, "cache8_store: null slots");
    rc = check_rows("cache8_store", k, k_stride, (int64_t)nkv * hs, half);
    if (!rc) rc = check_rows("cache8_store", v, v_stride, (int64_t)nkv * hs, half);
    if (rc) return rc;
    StoreArgs a = {{kc, vc}, {ks, vs}, {k, v}, {k_stride, v_stride}, slots, n, blocks, block, nkv, hs, 0};
    // Up to 512 tokens a warp each (and head), so that single ones are stored side by side; else a thread block for the runs
    // that begin among 16, which are few where prompts are stored. What tells the two apart is the runs' length, which only
    // the device knows; n stands for it. Measured (8 heads of 128, float32 and float16, by warps and by blocks): 64 single
    // tokens 3.3 and 4.9 us, 19 and 24; 512 of them 7.2 and 8.6, 27 and 30; 1024 12 and 14, 31 and 33. One prompt of 512
    // tokens 15 and 34, 6.7 and 6.6; of 1024 20 and 38, 8 and 12; 64 of 73 tokens 42 and 56, 20 and 23.
    if (n <= 512) {
      a.per = 1;
      launch(half ? cache8_store_kernel<true, 32> : cache8_store_kernel<false, 32>, dim3(n, (2 * nkv + 3) / 4), dim3(ST), 0,
             as_stream(stream), a);
    } else {
      a.per = 16;
      launch(half ? cache8_store_kernel<true, ST> : cache8_store_kernel<false, ST>, dim3((n + 15) / 16, 2 * nkv), dim3(ST), 0,
             as_stream(stream), a);
    }
    B200_LAUNCHED("cache8_store");
    return 0;
  } catch (...) {
    return fail(B200FWD_EINVAL, "cache8_store: exception");
  }
}

extern "C" int b200k_cache8_load(void *k, void *v, const int8_t *kc, const float *ks, const int8_t *vc,
                                 const float *vs, const int32_t *slots, int32_t n, int64_t k_stride, int64_t v_stride,
                                 int32_t blocks, int32_t block, int32_t nkv, int32_t hs, int32_t half,
                                 b200fwd_stream stream) {
  try {
    int rc = check_cache8("cache8_load", kc, ks, vc, vs, blocks, block, nkv, hs);
    if (rc) return rc;
    if (n < 0 || n > 1 << 30) return fail(B200FWD_EINVAL, "cache8_load: 0 to 2^30 tokens");
    if (n == 0) return 0;
    if (!slots) return fail(B200FWD_EINVAL, "cache8_load: null slots");
    rc = check_rows("cache8_load", k, k_stride, (int64_t)nkv * hs, half);
    if (!rc) rc = check_rows("cache8_load", v, v_stride, (int64_t)nkv * hs, half);
    if (rc) return rc;
    LoadArgs a = {{k, v}, {kc, vc}, {ks, vs}, {k_stride, v_stride}, slots, n, blocks, block, nkv, hs};
    const dim3 grid((n + L_TOKENS - 1) / L_TOKENS, (nkv * hs / (half ? 8 : 4) + LT - 1) / LT, 2);
    launch(half ? cache8_load_kernel<true> : cache8_load_kernel<false>, grid, dim3(LT), 0, as_stream(stream), a);
    B200_LAUNCHED("cache8_load");
    return 0;
  } catch (...) {
    return fail(B200FWD_EINVAL, "cache8_load: exception");
  }
}
