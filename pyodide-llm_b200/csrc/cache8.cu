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

// ------------------------------------------------------------------------------------------------ block tables
//
// L' = max(0, L + news) positions a request: its blocks go from ceil(L / block) to ceil(L' / block), new ones taken
// from the head of the ring of free ids in the requests' order, blocks left behind put at its tail. Bound by latency:
// a step of 64 requests moves 2 KB. So one launch does it all: one block, or one cluster of eight where there is more
// to write, and every block of the cluster adds up all requests by itself (8 bytes each, from L2) instead of waiting
// for partial sums. Takes read the ring's live part and gives write behind it, takes write table entries that no
// token's slot is read from (a token of a new block finds its id in the ring), so only lengths and state, which may
// be updated in place, have to wait until every block has read them: the one cluster barrier.

constexpr int TT = 512;  // threads, and the requests of one tile of the running sums

struct Need {
  int64_t tokens, take, give;
};

// what request i asks for; `bad` collects B200K_TABLES_* of requests that cannot have it
__device__ __forceinline__ Need need_of(int64_t length, int64_t add, int64_t most, int block, int &bad, int64_t &after) {
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
  const int before_b = (int)((length + block - 1) / block), after_b = (int)((after + block - 1) / block);
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
};

__global__ void __launch_bounds__(TT) block_tables_kernel(TablesArgs a) {
  pdl_begin();
  __shared__ int64_t part[3][TT / 32];
  __shared__ int bad_s, sums[3][TT + 1], len_s[TT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int64_t most = (int64_t)a.width * a.block;
  if (tid == 0) bad_s = 0;
  __syncthreads();

  // what everything comes to: all is granted, or nothing is
  int64_t sum[3] = {0, 0, 0};
  int bad = 0;
  for (int i = tid; i < a.n_seqs; i += TT) {
    int64_t after;
    const Need w = need_of(a.lengths[i], a.news[i], most, a.block, bad, after);
    sum[0] += w.tokens;
    sum[1] += w.take;
    sum[2] += w.give;
  }
#pragma unroll
  for (int j = 0; j < 3; j++) {
#pragma unroll
    for (int d = 16; d; d >>= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], d);
    if (lane == 0) part[j][warp] = sum[j];
  }
  if (bad) atomicOr(&bad_s, bad);
  const int head = a.state[0], count = a.state[1];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 3; j++) {
    sum[j] = 0;
    for (int w = 0; w < TT / 32; w++) sum[j] += part[j][w];
  }
  bad = bad_s;
  if (head < 0 || head >= a.blocks || count < 0 || count > a.blocks || count + sum[2] > a.blocks)
    bad |= 1 << B200K_TABLES_INPUT;
  if (sum[0] > a.n) bad |= 1 << B200K_TABLES_TOKENS;
  if (sum[1] > count) bad |= 1 << B200K_TABLES_BLOCKS;
  const bool granted = bad == 0;
  const int total = granted ? (int)sum[0] : 0;

  const int stride = (int)ranks * TT, first = (int)rank * TT + tid;
  int carry[3] = {0, 0, 0};
  if (granted) {
    for (int base = 0; base < a.n_seqs; base += TT) {
      const int i = base + tid, tile = min(TT, a.n_seqs - base);
      Need w = {0, 0, 0};
      int length = 0;
      if (i < a.n_seqs) {
        int64_t after;
        int none = 0;
        length = a.lengths[i];
        w = need_of(length, a.news[i], most, a.block, none, after);
      }
      int64_t run[3] = {w.tokens, w.take, w.give};
      __syncthreads();  // the tile before has been read
#pragma unroll
      for (int j = 0; j < 3; j++) {
        run[j] = warp_scan(run[j]);
        if (lane == 31) part[j][warp] = run[j];
      }
      len_s[tid] = length;
      __syncthreads();
      const int64_t own[3] = {w.tokens, w.take, w.give};
#pragma unroll
      for (int j = 0; j < 3; j++) {
        int64_t before = carry[j];
        for (int v = 0; v < warp; v++) before += part[j][v];
        sums[j][tid] = (int)(before + run[j] - own[j]);
        if (tid == TT - 1) sums[j][TT] = (int)(before + run[j]);
      }
      __syncthreads();
      if (tid < tile && rank == 0) a.starts[i] = sums[0][tid];
      // the tokens of this tile of requests, their slots from the table or, in blocks taken now, from the ring
      for (int t = carry[0] + first; t < sums[0][TT]; t += stride) {
        const int s = find(sums[0], tile, t), p = len_s[s] + (t - sums[0][s]), b = p / a.block;
        const int held = (len_s[s] + a.block - 1) / a.block;
        int id;
        if (b < held) {
          id = a.tables[(int64_t)(base + s) * a.width + b];
        } else {
          int64_t at = (int64_t)head + sums[1][s] + (b - held);
          id = a.ring[at % a.blocks];
        }
        a.slots[t] = id >= 0 && id < a.blocks ? id * a.block + (p - b * a.block) : -1;
        if (a.seq) a.seq[t] = base + s;
        if (a.pos) a.pos[t] = p;
      }
      for (int u = carry[1] + first; u < sums[1][TT]; u += stride) {
        const int s = find(sums[1], tile, u), held = (len_s[s] + a.block - 1) / a.block;
        a.tables[(int64_t)(base + s) * a.width + held + (u - sums[1][s])] = a.ring[((int64_t)head + u) % a.blocks];
      }
      for (int u = carry[2] + first; u < sums[2][TT]; u += stride) {
        const int s = find(sums[2], tile, u), held = (len_s[s] + a.block - 1) / a.block;
        // request s keeps its first held - (its gives) blocks
        const int gives = sums[2][s + 1] - sums[2][s];
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
  for (int t = total + first; t < a.n; t += stride) {
    a.slots[t] = -1;
    if (a.seq) a.seq[t] = -1;
    if (a.pos) a.pos[t] = -1;
  }
  // lengths and state may be updated in place: not before every block has read them
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
  for (int i = first; i < a.n_seqs; i += stride) {
    int64_t after = a.lengths[i];
    if (granted) {
      int none = 0;
      need_of(after, a.news[i], most, a.block, none, after);
    }
    a.lengths_out[i] = (int)after;
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

// ------------------------------------------------------------------------------------------------------- store
//
// A (block, head)'s scale is s = max |x| / 127 in float32 over all that it holds, and every value is the integer
// nearest to x / s, half to even, of the real quotient: a float32 guess, then the exact remainder decides. A token
// that raises the scale of a block with earlier tokens in it has their integers q brought to the new step,
// nearest(q s_old / s): one scale a block costs that, and only blocks that a request still fills pay it.
//
// Tokens of a block stand together in the call (a request's positions do), so the block's work belongs to the place
// where its run of tokens begins: no two thread blocks touch one (block, head), and no atomics.

constexpr int ST = 128;  // threads
constexpr int KEEP = 8;  // 16-byte vectors of new values that a thread keeps in registers between its two passes

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

// the integer nearest to x / s (half to even), |x| <= 127 s (1 + 2^-24), inv about 1 / s
__device__ __forceinline__ int nearest(float x, float s, float inv) {
  float q = rintf(__fmul_rn(x, inv));
  // x - q s is exact: a multiple of s's last place, and no larger than about s
  const float r = __fmaf_rn(-q, s, x);
  const float twice = __fadd_rn(fabsf(r), fabsf(r));
  if (twice > s) {
    q = __fadd_rn(q, r > 0 ? 1.0f : -1.0f);
  } else if (twice == s) {
    // halfway between q and its neighbour on r's side: the even one
    if ((int)q & 1) q = __fadd_rn(q, r > 0 ? 1.0f : -1.0f);
  }
  return (int)q;
}

// nearest(q a / b), a <= b, in 64 bits (q a is exact there, the quotient's halves too): few values need it
__device__ __forceinline__ int moved(int q, double a, double b) { return (int)rint(__ddiv_rn(__dmul_rn((double)q, a), b)); }

// the largest |x| as its bits: NaN above infinity above every number, so the maximum keeps both
template <int VW>
__device__ __forceinline__ uint32_t largest_bits(const uint4 &u) {
  float x[VW];
  values_of(u, x);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VW; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

template <int VW>
__device__ __forceinline__ void put(int8_t *dst, const uint4 &u, float s, float inv) {
  float x[VW];
  values_of(u, x);
  uint32_t w[VW / 4];
#pragma unroll
  for (int i = 0; i < VW / 4; i++) {
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      // s 0: the block holds zeros (or values under half a step of the smallest float); s NaN: it held none
      const int q = s > 0 ? nearest(x[4 * i + j], s, inv) : 0;
      b |= (uint32_t)(q & 255) << (8 * j);
    }
    w[i] = b;
  }
  if (VW == 8) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[VW / 4 - 1]);
  else *reinterpret_cast<uint32_t *>(dst) = w[0];
}

struct StoreArgs {
  int8_t *cache[2];
  float *scales[2];
  const void *x[2];
  int64_t stride[2];
  const int32_t *slots;
  int n, blocks, block, nkv, hs, per;
};

template <bool HALF>
__global__ void __launch_bounds__(ST) cache8_store_kernel(StoreArgs a) {
  pdl_begin();
  constexpr int VW = HALF ? 8 : 4;  // values of a 16-byte vector
  __shared__ uint32_t top[ST / 32];
  const int tid = threadIdx.x, h = blockIdx.y;
  const bool second = blockIdx.z;  // keys, then values
  int8_t *cache = second ? a.cache[1] : a.cache[0];
  float *scales = second ? a.scales[1] : a.scales[0];
  const char *x = reinterpret_cast<const char *>(second ? a.x[1] : a.x[0]);
  const int64_t stride = second ? a.stride[1] : a.stride[0];
  const int vpr = a.hs / VW, rows = ST / vpr, row = tid / vpr, col = (tid % vpr) * VW;
  const int i0 = blockIdx.x * a.per, i1 = min(a.n, i0 + a.per), lane = tid & 31;
  // the block of token i, or -1 (every warp looks the slots over by itself, a lane a token)
  auto page_of = [&](int i) {
    const int slot = i >= 0 && i < a.n ? a.slots[i] : -1, page = slot / a.block;
    return slot >= 0 && page < a.blocks ? page : -1;
  };
  const int mine = i0 + lane < i1 ? page_of(i0 + lane) : -1;
  uint32_t begins = __ballot_sync(0xffffffffu, mine >= 0 && mine != page_of(i0 + lane - 1));
  for (; begins; begins &= begins - 1) {
    const int i = i0 + __ffs(begins) - 1, page = __shfl_sync(0xffffffffu, mine, i - i0), slot = a.slots[i];
    int m = 1;  // the run of tokens of this block
    for (;;) {
      const uint32_t other = __ballot_sync(0xffffffffu, page_of(i + m + lane) != page);
      if (other) {
        m += __ffs(other) - 1;
        break;
      }
      m += 32;
    }
    const int held = slot - page * a.block;  // earlier tokens in the block
    int8_t *dst = cache + ((int64_t)page * a.nkv + h) * a.block * a.hs;
    float *scale = scales + (int64_t)page * a.nkv + h;
    const float s_old = held ? *scale : 0.0f;
    const char *src = x + ((int64_t)i * stride + (int64_t)h * a.hs + col) * (HALF ? 2 : 4);
    const int64_t step = stride * (HALF ? 2 : 4);
    uint4 kept[KEEP];
    uint32_t bits = 0;
    if (row < rows) {
#pragma unroll
      for (int u = 0; u < KEEP; u++) {
        const int t = row + u * rows;
        if (t < m) kept[u] = *reinterpret_cast<const uint4 *>(src + t * step);
      }
#pragma unroll
      for (int u = 0; u < KEEP; u++)
        if (row + u * rows < m) bits = max(bits, largest_bits<VW>(kept[u]));
      for (int t = row + KEEP * rows; t < m; t += rows)
        bits = max(bits, largest_bits<VW>(*reinterpret_cast<const uint4 *>(src + t * step)));
    }
    bits = __reduce_max_sync(0xffffffffu, bits);
    __syncthreads();  // the run before has read its maximum (and, in place, its scale)
    if ((tid & 31) == 0) top[tid >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < ST / 32; w++) bits = max(bits, top[w]);
    // a value that is no finite number, now or among the earlier ones, makes the block's scale NaN: its values read
    // as NaN until the block is begun again
    float s = bits < 0x7f800000u ? __fdiv_rn(__uint_as_float(bits), 127.0f) : __uint_as_float(0x7fffffffu);
    if (!(s_old <= s)) s = s != s ? s : s_old;
    const float inv = s > 1e-37f ? __fdiv_rn(1.0f, s) : 0.0f;
    if (tid == 0) *scale = s;
    if (s > s_old && s_old > 0) {
      // the earlier tokens' integers to the new step
      const int words = held * a.hs / 4;
      uint32_t *q4 = reinterpret_cast<uint32_t *>(dst);
      for (int w = tid; w < words; w += ST) {
        const uint32_t q = q4[w];
        uint32_t b = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) b |= (uint32_t)(moved((int8_t)(q >> (8 * j)), s_old, s) & 255) << (8 * j);
        q4[w] = b;
      }
    }
    if (row < rows) {
      // a scale so small that its inverse is no float: its values over the scale brought into range first
      const bool tiny = s > 0 && !(s > 1e-37f);
      auto one = [&](int t, uint4 v) {
        const int at = a.slots[i + t] - page * a.block;
        if (tiny) {
          float y[VW];
          values_of(v, y);
#pragma unroll
          for (int j = 0; j < VW; j++) dst[at * a.hs + col + j] = (int8_t)moved(1, y[j], s);
        } else {
          put<VW>(dst + at * a.hs + col, v, s, inv);
        }
      };
#pragma unroll
      for (int u = 0; u < KEEP; u++)
        if (row + u * rows < m) one(row + u * rows, kept[u]);
      for (int t = row + KEEP * rows; t < m; t += rows) one(t, *reinterpret_cast<const uint4 *>(src + t * step));
    }
  }
}

// -------------------------------------------------------------------------------------------------------- load
//
// q s, rounded once to the output's type. Bound by its writes (4 or 2 bytes a value for the 1 read): a thread keeps
// its columns for several tokens and writes 16 bytes a token.

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
    const int page = slot[t] / a.block, at = slot[t] - page * a.block;
    const int64_t ph = (int64_t)page * a.nkv + h;
    const int8_t *src = cache + (ph * a.block + at) * a.hs + col;
    if (HALF) q[t] = *reinterpret_cast<const uint2 *>(src);
    else q[t].x = *reinterpret_cast<const uint32_t *>(src);
    s[t] = scales[ph];
  }
#pragma unroll
  for (int t = 0; t < L_TOKENS; t++) {
    if (slot[t] < 0) continue;
    float x[VW];
#pragma unroll
    for (int j = 0; j < VW; j++) x[j] = __fmul_rn((float)(int8_t)((j < 4 ? q[t].x : q[t].y) >> (8 * (j & 3))), s[t]);
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
        (int64_t)table_width * block > INT32_MAX)
      return fail(B200FWD_EINVAL, "block_tables: 1 block at least, and positions and slots that an int32 holds");
    TablesArgs a = {tables, ring, state_out, lengths_out, starts, slots, seq, pos, state, lengths, news,
                    n_seqs, table_width, blocks, block, n};
    // one block up to 4096 tokens and 2 tiles of requests, else a cluster of eight
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
    a.per = n <= 256 ? 1 : n <= 2048 ? 4 : 16;
    const dim3 grid((n + a.per - 1) / a.per, nkv, 2);
    launch(half ? cache8_store_kernel<true> : cache8_store_kernel<false>, grid, dim3(ST), 0, as_stream(stream), a);
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
