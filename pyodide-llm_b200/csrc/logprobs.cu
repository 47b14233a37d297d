// logprobs.cu — b200k_logprobs: of each row of logits the log probability of a given token, the entropy and the k most
// probable tokens with theirs: log p_j = (x_j - m) - log S, S = sum exp(x - m), H = log S - sum e (x - m) / S.
//
// Bound by reading the logits once. A row belongs to a cluster of 1 to 8 thread blocks, each with a slice of it that
// its threads stream through rings of their own in shared memory (cp.async, 12 vectors of 16 bytes deep; a thread reads
// back only what it copied, so none waits for another) with a running maximum and sums a thread. The clusters go from
// row to row, and the rings run ahead into the next row while a row's results are put together.
// The k largest: of the 4 largest thread maxima of each of a block's 8 warps the k-th is a bound: at least k values are
// no smaller, and hardly more are. Threads whose maximum reaches it (about k) read the group of vectors that it came
// from once more, from L2 (all their groups, where a second one reaches it too), and list what does, to be ranked by
// (value, lowest id). Values equal to the bound, which may be thousands (masks), have a list of their own; where it
// runs over, the lowest ids among them are looked for in order. Where few threads hold nearly all the largest values
// and the first list runs over, the k are picked one after the other.
// A row's partial results meet in one block of its cluster, a different one from row to row, which adds them in the
// blocks' order while the others go on (the cluster's barrier is waited for a row later).
// Measured at 128256 float32 logits: 512 rows 53 us without alternatives (4.9 TB/s, 0.75 of a copy's rate), 63 us with
// 20; 64 rows 11 and 16 us, of which a row's chain of exchanges is most. One row of 1024: 3.6 and 6.2 us.
#include <cuda_fp16.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

#include "common.h"

namespace b200 {
namespace {

constexpr int T = 256, WARPS = T / 32;
// Blocks of an SM: with two a thread has 128 registers and nothing spills; 512 rows of 128256 logits took 54 us so, 63 us
// with three (80 registers), 66 us with four.
constexpr int RESIDENT = 2;
constexpr int K_MOST = 32;
constexpr int LIST = 512, EQUAL = 128;  // values that a block lists of a row: above the bound, and equal to it
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct Args {
  float *logprob, *entropy, *top;
  int32_t *ids;
  const void *x;
  const int32_t *targets;
  int64_t stride;
  int count, n, k;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t fma_2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul_2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add_2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

__device__ __forceinline__ void values_of(const uint4 &u, float (&y)[4]) {
  y[0] = __uint_as_float(u.x), y[1] = __uint_as_float(u.y), y[2] = __uint_as_float(u.z), y[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void values_of(const uint4 &u, float (&y)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    y[2 * i] = f.x, y[2 * i + 1] = f.y;
  }
}

// floats in the order of unsigned integers (-0 as 0), and back; 0 is below every float
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}
// larger values first, equal ones by the lowest id
__device__ __forceinline__ uint64_t entry_of(uint32_t key, int id) { return ((uint64_t)key << 32) | (uint32_t)~id; }

struct Out {  // a block's results of a row
  float m, S, Te;
  uint64_t best[K_MOST];
};
struct Smem {
  float sums[2][WARPS];
  uint32_t top[WARPS][4], low[WARPS], part[WARPS];
  uint64_t list[LIST], equal[EQUAL], picked[WARPS];  // (list: in the finisher then every block's best)
  int found[WARPS];
  // By turns: a block may be filling one for row t while the finisher of row t - 2 still reads (it arrives at the barrier
  // of row t - 1 after that, and that is waited for only at row t's end); the one of row t - 3 has been read.
  Out out[3];
  int listed[3], equals[3];
};

__device__ __forceinline__ void copy_vector(uint32_t dst, const uint4 *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// a shared variable's counterpart in the cluster's block `rank`
template <typename V>
__device__ __forceinline__ V peer(const V *p, uint32_t rank) {
  const uint32_t local = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(local), "r"(rank));
  if constexpr (sizeof(V) == 8) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return (V)v;
  } else {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return __uint_as_float(v);
  }
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

constexpr int GROUP = 4, GROUPS = 4;  // vectors of 16 bytes that a thread copies at a time, and how often it does ahead

template <bool HALF>
__global__ void __launch_bounds__(T, RESIDENT) logprobs_kernel(const Args a) {
  pdl_begin();
  constexpr int VW = HALF ? 8 : 4;
  __shared__ Smem sm;
  extern __shared__ __align__(16) uint4 ring[];  // [GROUPS][GROUP][T]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int clusters = gridDim.x / ranks;
  using E = typename std::conditional<HALF, __half, float>::type;

  // a row: whole vectors from the first 16-byte boundary on, of which this thread has v0, v0 + T, ... below v1; the few
  // values before and behind them are the first block's
  struct Row {
    const E *x;
    int lead, vecs, slice, v0, v1;
  };
  auto row_of = [&](int row) {
    Row r;
    r.x = reinterpret_cast<const E *>(a.x) + (int64_t)row * a.stride;
    r.lead = min(a.n, (int)(((16 - (reinterpret_cast<uintptr_t>(r.x) & 15)) & 15) / sizeof(E)));
    r.vecs = (a.n - r.lead) / VW;
    const int per = (r.vecs + (int)ranks - 1) / (int)ranks;
    r.v0 = min(r.vecs, (int)rank * per) + tid;
    r.v1 = min(r.vecs, ((int)rank + 1) * per);
    r.slice = r.v1 - (r.v0 - tid);
    return r;
  };
  // the ring's front: the next group to copy, `left` vectors of the row at and behind front_src (for thread 0)
  int front_row = blockIdx.x / ranks, front_left;
  const uint4 *front_src;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring + tid));
  uint32_t front_at = ring_at;
  auto front_begin = [&]() {
    const Row r = row_of(front_row < a.count ? front_row : 0);
    front_src = reinterpret_cast<const uint4 *>(r.x + r.lead) + r.v0;
    front_left = r.slice;
  };
  front_begin();
  auto copy_group = [&]() {
    if (front_row < a.count) {
      if (front_left >= GROUP * T) {
#pragma unroll
        for (int i = 0; i < GROUP; i++) copy_vector(front_at + i * T * 16, front_src + i * T);
      } else {
        for (int i = 0; tid + i * T < front_left; i++) copy_vector(front_at + i * T * 16, front_src + i * T);
      }
      front_src += GROUP * T;
      front_left -= GROUP * T;
      if (front_left <= 0) {
        front_row += clusters;
        front_begin();
      }
      front_at = front_at == ring_at + (GROUPS - 1) * GROUP * T * 16 ? ring_at : front_at + GROUP * T * 16;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int g = 0; g < GROUPS; g++) copy_group();

  int slot = 0, turn = 0;
  bool pending = false;  // arrived at the cluster's barrier, not waited
  if (tid == 0) sm.listed[0] = sm.equals[0] = 0;
  const uint64_t l2 = f2(LOG2E, LOG2E);
  for (int row = blockIdx.x / ranks; row < a.count; row += clusters, turn = turn == 2 ? 0 : turn + 1) {
    const Row r = row_of(row);
    Out &out = sm.out[turn];
    const uint32_t finisher = (row / clusters) % ranks;
    float x_target = __uint_as_float(0x7fffffffu);
    if (tid == 0 && rank == finisher && a.logprob) {
      const int t = a.targets[row];
      if (t >= 0 && t < a.n) x_target = (float)r.x[t];
    }
    float edge = -INFINITY;  // the odd value of this thread
    int edge_id = -1;
    if (rank == 0) {
      const int tail = r.lead + r.vecs * VW;
      if (tid < r.lead) edge_id = tid;
      else if (tid >= 32 && tail + tid - 32 < a.n) edge_id = tail + tid - 32;
      if (edge_id >= 0) edge = (float)r.x[edge_id];
    }
    // This thread's maximum, its groups' second and third largest maxima, the groups of the first two; its sums (by halves)
    // of e = 2^d and of e d, d = (x - from) log2 e, from: a maximum that the running one passed by no more than 8 (so the
    // sums are hardly ever rescaled; a lone value's e is 1 exactly)
    float m = edge, second = -INFINITY, third = -INFINITY, from = edge;
    int best_group = 0, second_group = 0;
    uint64_t s2 = f2(edge > -INFINITY ? 1.0f : 0.0f, 0.0f), t2 = f2(0.0f, 0.0f);
    auto raise = [&](float most, int g) {
      const float less = fminf(m, most);
      const int less_group = most > m ? best_group : g;
      if (most > m) best_group = g;
      third = fmaxf(third, fminf(second, less));
      if (less > second) second_group = less_group;
      second = fmaxf(second, less);
      m = max_nan(m, most);
      if (most > from + 8.0f) {
        const float d = (from - most) * LOG2E, by = from == -INFINITY ? 0.0f : ex2(d);
        t2 = by == 0.0f ? f2(0.0f, 0.0f) : mul_2(fma_2(s2, f2(d, d), t2), f2(by, by));
        s2 = mul_2(s2, f2(by, by));
        from = most;
      }
    };
    // (a slice of no vectors has a group too: the front's does)
    for (int left = r.slice, g = 0;; g++) {
      asm volatile("cp.async.wait_group %0;" ::"n"(GROUPS - 1) : "memory");
      const uint4 *own = ring + slot * GROUP * T + tid;
      bool slow = left < GROUP * T;
      if (!slow) {
        uint4 u[GROUP];
#pragma unroll
        for (int i = 0; i < GROUP; i++) u[i] = own[i * T];
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < GROUP; i++) {
          float y[VW];
          values_of(u[i], y);
#pragma unroll
          for (int j = 0; j < VW; j += 2) most = max3(most, y[j], y[j + 1]);
        }
        raise(most, g);
        const uint64_t m2 = f2(-from, -from);
        uint64_t s_new = s2, t_new = t2;
#pragma unroll
        for (int i = 0; i < GROUP; i++) {
          float y[VW];
          values_of(u[i], y);
#pragma unroll
          for (int j = 0; j < VW; j += 2) {
            const uint64_t d = mul_2(add_2(f2(y[j], y[j + 1]), m2), l2);
            const uint64_t e = f2(ex2(lo_of(d)), ex2(hi_of(d)));
            s_new = add_2(s_new, e);
            t_new = fma_2(e, d, t_new);
          }
        }
        // 0 times -inf, or a NaN among the values
        const float test = lo_of(t_new) + hi_of(t_new);
        if (test == test) s2 = s_new, t2 = t_new;
        else slow = true;
      }
      if (slow) {
        // the row's last vectors, or a masked part: vector by vector, d held above -1e4, where e is 0 and e d too
        float most = -INFINITY;
#pragma unroll 1
        for (int i = 0; i < GROUP && tid + i * T < left; i++) {
          float y[VW];
          values_of(own[i * T], y);
#pragma unroll
          for (int j = 0; j < VW; j++) most = max_nan(most, y[j]);
        }
        if (left < GROUP * T) raise(most, g);
        m = max_nan(m, most);
        const uint64_t m2 = f2(-from, -from);
#pragma unroll 1
        for (int i = 0; i < GROUP && tid + i * T < left && most > -INFINITY; i++) {
          float y[VW];
          values_of(own[i * T], y);
#pragma unroll
          for (int j = 0; j < VW; j += 2) {
            const uint64_t d = mul_2(add_2(f2(y[j], y[j + 1]), m2), l2);
            const float d0 = fmaxf(lo_of(d), -1e4f), d1 = fmaxf(hi_of(d), -1e4f);
            const uint64_t e = f2(ex2(d0), ex2(d1));
            s2 = add_2(s2, e);
            t2 = fma_2(e, f2(d0, d1), t2);
          }
        }
      }
      copy_group();
      slot = slot + 1 == GROUPS ? 0 : slot + 1;
      left -= GROUP * T;
      if (left <= 0) break;
    }
    float S = lo_of(s2) + hi_of(s2), Te = lo_of(t2) + hi_of(t2);

    // ---- the block's maximum and sums; the bound of the k largest
    const int full = min(WARPS, r.slice / 32);  // warps whose threads all have values
    const uint32_t key = r.v0 < r.v1 || edge_id >= 0 ? key_of(m) : 0;
    {
      uint32_t rest = key, top = __reduce_max_sync(0xffffffffu, key);
      if (lane == 0) sm.part[warp] = top;
      if (tid == 0) sm.listed[turn == 2 ? 0 : turn + 1] = sm.equals[turn == 2 ? 0 : turn + 1] = 0;
      if (a.k) {
        // (a slice of few values: the full warps' ceil(k / full)-th)
        const int most = full == WARPS ? 4 : full ? (a.k + full - 1) / full : 0;
        for (int j = 0; j < most; j++) {
          if (j) top = __reduce_max_sync(0xffffffffu, rest);
          const uint32_t holds = __ballot_sync(0xffffffffu, rest == top);
          if (lane == __ffs(holds) - 1) rest = 0;
          if (lane == 0 && j < 4) sm.top[warp][j] = top;
        }
        if (lane == 0) sm.low[warp] = top;
      }
    }
    __syncthreads();
    uint32_t block_key = sm.part[0];
#pragma unroll
    for (int w = 1; w < WARPS; w++) block_key = max(block_key, sm.part[w]);
    const float block_m = block_key ? value_of(block_key) : -INFINITY;
    int *listed_s = &sm.listed[turn], *equals_s = &sm.equals[turn];
    float floor = -INFINITY;
    if (a.k) {
      uint32_t low = 0;
      if (full == WARPS) {
        const uint32_t mine = sm.top[lane >> 2][lane & 3];
        int better = 0;
#pragma unroll
        for (int j = 1; j < 32; j++) {
          const uint32_t other = __shfl_sync(0xffffffffu, mine, (lane + j) & 31);
          better += other > mine || (other == mine && ((lane + j) & 31) < lane);
        }
        low = __reduce_max_sync(0xffffffffu, better == a.k - 1 ? mine : 0);
      } else if (full) {
        low = 0xffffffffu;
        for (int w = 0; w < full; w++) low = min(low, sm.low[w]);
      }
      if (low) floor = value_of(low);
      auto list = [&](float y, int id) {
        if (y > floor) {
          const int at = atomicAdd(listed_s, 1);
          if (at < LIST) sm.list[at] = entry_of(key_of(y), id);
        } else if (y == floor && *(volatile int *)equals_s <= EQUAL) {
          const int at = atomicAdd(equals_s, 1);
          if (at < EQUAL) sm.equal[at] = entry_of(key_of(y), id);
        }
      };
      const uint4 *src = reinterpret_cast<const uint4 *>(r.x + r.lead);
      const bool reaches = key && key >= low;
      const int groups = !reaches ? 0 : second >= floor && second_group != best_group ? 2 : 1;
#pragma unroll 1
      for (int g = 0; g < groups; g++) {
        const int v = r.v0 + (g ? second_group : best_group) * GROUP * T;
        uint4 u[GROUP];
#pragma unroll
        for (int i = 0; i < GROUP; i++)
          if (v + i * T < r.v1) u[i] = src[v + i * T];
#pragma unroll
        for (int i = 0; i < GROUP; i++)
          if (v + i * T < r.v1) {
            float y[VW];
            values_of(u[i], y);
#pragma unroll
            for (int j = 0; j < VW; j++)
              if (y[j] >= floor) list(y[j], r.lead + (v + i * T) * VW + j);
          }
      }
      if (reaches && edge_id >= 0) list(edge, edge_id);
      // the other groups of a thread with a third one: its warp reads them together (values equal to the bound only as long
      // as their list has room: past it they are looked for in order)
      __syncwarp();
      auto wanted = [&](float y) { return y > floor || (y == floor && *(volatile int *)equals_s <= EQUAL); };
      for (uint32_t more = __ballot_sync(0xffffffffu, reaches && wanted(third)); more; more &= more - 1) {
        const int whose = __ffs(more) - 1;
        const int first = __shfl_sync(0xffffffffu, best_group, whose), then = __shfl_sync(0xffffffffu, second_group, whose);
        const int v0 = r.v0 - lane + whose;
#pragma unroll 4
        for (int i = lane; v0 + i * T < r.v1; i += 32) {
          float y[VW], most = -INFINITY;
          values_of(src[v0 + i * T], y);
#pragma unroll
          for (int j = 0; j < VW; j++) most = fmaxf(most, y[j]);
          if (wanted(most) && i / GROUP != first && i / GROUP != then)
#pragma unroll 1
            for (int j = 0; j < VW; j++) list((float)r.x[r.lead + (v0 + i * T) * VW + j], r.lead + (v0 + i * T) * VW + j);
        }
      }
    }
    if (from != block_m) {
      const float d = (from - block_m) * LOG2E, by = from == -INFINITY ? 0.0f : ex2(d);
      Te = by == 0.0f ? 0.0f : (Te + S * d) * by;
      S *= by;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      S += __shfl_xor_sync(0xffffffffu, S, d);
      Te += __shfl_xor_sync(0xffffffffu, Te, d);
    }
    if (lane == 0) sm.sums[0][warp] = S, sm.sums[1][warp] = Te;
    __syncthreads();

    // ---- the block's k largest
    int listed = a.k ? *listed_s : 0;
    const int equals = a.k ? *equals_s : 0;
    // this block's values in the order of their ids (the first block's last few follow its slice)
    const int begin = r.v0 - tid, values = (r.v1 - begin) * VW, ahead = rank == 0 ? r.lead : 0;
    const int length = ahead + values + (rank == 0 ? a.n - r.lead - r.vecs * VW : 0);
    auto id_of = [&](int q) {
      return q < ahead + values ? r.lead - ahead + begin * VW + q : r.lead + r.vecs * VW + q - ahead - values;
    };
    if (listed > LIST) {
      // one after the other: the largest below the one picked last
      uint64_t last = ~0ull;
      for (listed = 0; listed < a.k; listed++) {
        uint64_t pick = 0;
        for (int q = tid; q < length; q += T) {
          const uint64_t e = entry_of(key_of((float)r.x[id_of(q)]), id_of(q));
          if (e < last && e > pick) pick = e;
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
          const uint64_t o = __shfl_xor_sync(0xffffffffu, pick, d);
          if (o > pick) pick = o;
        }
        __syncthreads();
        if (lane == 0) sm.picked[warp] = pick;
        __syncthreads();
        for (int w = 0; w < WARPS; w++)
          if (sm.picked[w] > pick) pick = sm.picked[w];
        if (!pick) break;
        last = pick;
        if (tid == 0) sm.list[listed] = pick;
      }
    } else if (listed < a.k && equals <= EQUAL) {
      if (tid < equals) sm.list[listed + tid] = sm.equal[tid];
      listed += equals;
    } else if (listed < a.k) {
      // the lowest ids among the values equal to the bound
      for (int q0 = 0; q0 < length && listed < a.k; q0 += T) {
        const int q = q0 + tid;
        const bool is = q < length && (float)r.x[id_of(q)] == floor;
        const uint32_t holds = __ballot_sync(0xffffffffu, is);
        __syncthreads();
        if (lane == 0) sm.found[warp] = __popc(holds);
        __syncthreads();
        int at = listed + __popc(holds & ((1u << lane) - 1));
        for (int w = 0; w < warp; w++) at += sm.found[w];
        if (is && at < a.k) sm.list[at] = entry_of(key_of(floor), id_of(q));
        for (int w = 0; w < WARPS; w++) listed += sm.found[w];
      }
      listed = min(listed, a.k);
    }
    __syncthreads();
    for (int i = tid; i < listed; i += T) {
      const uint64_t e = sm.list[i];
      int better = 0;
#pragma unroll 4
      for (int j = 0; j < listed; j++) better += sm.list[j] > e;
      if (better < a.k) out.best[better] = e;
    }
    if (tid >= listed && tid < a.k) out.best[tid] = 0;
    if (tid == 0) {
      S = Te = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; w++) S += sm.sums[0][w], Te += sm.sums[1][w];
      out.m = block_m, out.S = S, out.Te = Te;
    }
    if (ranks > 1) {
      __syncwarp();
      if (pending) cluster_wait();
      cluster_arrive();
      pending = rank != finisher;
      if (pending) continue;
      cluster_wait();
    } else {
      __syncthreads();
    }
    float M = -INFINITY, sum = 0.0f, dot = 0.0f;
    {
      float pm[8], ps[8], pt[8];
#pragma unroll
      for (int q = 0; q < 8; q++)
        if (q < (int)ranks) pm[q] = peer(&out.m, q), ps[q] = peer(&out.S, q), pt[q] = peer(&out.Te, q);
      if (tid < (int)ranks * a.k) sm.list[tid] = peer(&out.best[tid % a.k], tid / a.k);
#pragma unroll
      for (int q = 0; q < 8; q++)
        if (q < (int)ranks) M = max_nan(M, pm[q]);
#pragma unroll
      for (int q = 0; q < 8; q++)
        if (q < (int)ranks && pm[q] != -INFINITY) {
          const float d = (pm[q] - M) * LOG2E, by = ex2(d);
          sum += ps[q] * by;
          if (by != 0.0f) dot += (pt[q] + ps[q] * d) * by;
        }
    }
    __syncthreads();
    // no finite largest logit (all masked, an infinity, a NaN): no distribution
    const bool fine = fabsf(M) < INFINITY;
    const float logS = fine ? logf(sum) : __uint_as_float(0x7fffffffu);
    // (from sums of rounded terms: no log probability is above 0)
    auto logp = [&](float x) {
      const float l = (x - M) - logS;
      return l > 0.0f ? 0.0f : l;
    };
    if (tid == 0) {
      if (a.logprob) a.logprob[row] = logp(x_target);
      if (a.entropy) a.entropy[row] = logS - __fdiv_rn(dot, sum) * LN2;
    }
    if (!fine) {
      if (tid < a.k) {
        a.ids[(int64_t)row * a.k + tid] = -1;
        a.top[(int64_t)row * a.k + tid] = logS;
      }
    } else if (tid < (int)ranks * a.k) {
      // its place: the entries of every block's list, largest first, that are larger
      const uint64_t e = sm.list[tid];
      int at[8], better = 0;
#pragma unroll
      for (int q = 0; q < 8; q++) at[q] = 0;
#pragma unroll
      for (int step = K_MOST; step; step >>= 1)
#pragma unroll
        for (int q = 0; q < 8; q++)
          if (q < (int)ranks && at[q] + step <= a.k && sm.list[q * a.k + at[q] + step - 1] > e) at[q] += step;
#pragma unroll
      for (int q = 0; q < 8; q++) better += at[q];
      if (e && better < a.k) {
        const int64_t place = (int64_t)row * a.k + better;
        a.ids[place] = ~(int)(uint32_t)e;
        a.top[place] = logp(value_of((uint32_t)(e >> 32)));
      }
    }
    __syncthreads();  // sm.list has been read
  }
  if (ranks > 1) {
    // no block leaves while the last row's finisher may read its shared memory
    if (pending) cluster_wait();
    cluster_arrive();
    cluster_wait();
  }
}

template <bool HALF>
int launch_logprobs(const Args &a, int count, cudaStream_t stream) {
  constexpr int VW = HALF ? 8 : 4;
  auto kernel = logprobs_kernel<HALF>;
  constexpr int smem = GROUPS * GROUP * T * 16;
  // Blocks of a row: one where the rows fill the GPU (a block's work on a row beyond its values is then done once), more
  // while the GPU has room for all rows' blocks and a thread more than one vector. Measured (128256 float32 logits, k 5): a
  // row by one block 18.1 us, by eight 9.8; 64 rows by one 19.4, by four 14.1, by eight 21.3; 148 by one 19.5, by two 18.7,
  // by four 31.3. (37 rows by eight take 19.5, by one 18.8: 32 clusters of eight are resident at once.)
  const int vecs = (a.n + VW - 1) / VW;
  int ranks = 1;
  while (ranks < 8 && count * ranks * 2 <= 148 * RESIDENT && vecs > ranks * T) ranks *= 2;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(T);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_on() ? 2 : 1;
  B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  // as many clusters as are resident at once (a cluster stays within one of the GPU's partitions of SMs, so not every
  // SM takes its four blocks), or the rows
  static std::atomic<int> resident[9];  // by ranks (the same for every B200)
  int clusters = resident[ranks].load(std::memory_order_relaxed);
  if (clusters < 1) {
    cfg.gridDim = dim3(ranks);
    B200_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
    if (clusters < 1) clusters = 1;
    resident[ranks].store(clusters, std::memory_order_relaxed);
  }
  cfg.gridDim = dim3((unsigned)(count < clusters ? count : clusters) * ranks);
  (void)cudaLaunchKernelEx(&cfg, kernel, a);
  B200_LAUNCHED("logprobs");
  return 0;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200k_logprobs(float *logprob, float *entropy, float *top_logprob, int32_t *top_id, const void *logits,
                              const int32_t *targets, int32_t count, int32_t n, int64_t stride, int32_t k,
                              int32_t half, b200fwd_stream stream) {
  try {
    if (count < 0 || count > 1 << 24) return fail(B200FWD_EINVAL, "logprobs: 0 to 2^24 rows");
    if (n < 1 || n > 1 << 30 || stride < n) return fail(B200FWD_EINVAL, "logprobs: rows of 1 to 2^30 logits, a stride no smaller");
    if (k < 0 || k > K_MOST || k > n) return fail(B200FWD_EINVAL, "logprobs: 0 to 32 alternatives, no more than logits");
    if (!logits || (logprob && !targets) || (k > 0 && (!top_logprob || !top_id)))
      return fail(B200FWD_EINVAL, "logprobs: null pointer");
    if (reinterpret_cast<uintptr_t>(logits) % (half ? 2 : 4)) return fail(B200FWD_EINVAL, "logprobs: misaligned logits");
    if (count == 0) return 0;
    const Args a = {logprob, entropy, top_logprob, top_id, logits, targets, stride, count, n, k};
    return half ? launch_logprobs<true>(a, count, as_stream(stream)) : launch_logprobs<false>(a, count, as_stream(stream));
  } catch (...) {
    return fail(B200FWD_EINVAL, "logprobs: exception");
  }
}
