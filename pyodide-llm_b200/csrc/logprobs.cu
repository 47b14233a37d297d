// logprobs.cu — b200k_logprobs: of each row of logits the log probability of a given token, the entropy and the k most
// probable tokens with theirs: log p_j = (x_j - m) - log S, S = sum exp(x - m), H = log S - sum e (x - m) / S.
//
// Bound by reading the logits once. A row belongs to a cluster of 1 to 8 thread blocks, each with a slice of it that
// its threads hold in registers (up to 64 values a thread, all loads in flight at once), so the maximum is known
// before the first exponential, and the k largest are sought among registers, not by another pass over memory. Slices
// longer than that (rows of more than 131,072 logits) go round by round, with the sums rescaled and the best k so far
// kept. Partial results meet in the first block's shared memory; it adds them in the blocks' order.
// The k largest of a round: each of the 8 warps takes its ceil(k / 8)-th largest thread maximum, so at least k values
// are no smaller than the least of these; the values above it (and above the k-th of earlier rounds) are listed, a few
// dozen as a rule, and ranked against one another by (value, lowest id). Where too many are equal or a few threads
// hold them all, the list overflows and the round picks its k one after the other instead.
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "common.h"

namespace b200 {
namespace {

constexpr int T = 256, WARPS = T / 32;
constexpr int K_MOST = 32;
constexpr int LIST = 512;  // listed values of a round

struct Args {
  float *logprob, *entropy, *top;
  int32_t *ids;
  const void *x;
  const int32_t *targets;
  int64_t stride;
  int n, k;
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

struct Smem {
  float part[3][WARPS];
  uint32_t low[WARPS];
  uint64_t list[LIST], best[K_MOST], picked[WARPS];
  uint64_t all[8 * K_MOST];
  float mst[3];
  int count;
};

// block-wide reductions, every thread gets the result
__device__ __forceinline__ float block_max(float v, float *part) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < WARPS; w++) v = max_nan(v, part[w]);
  return v;
}

// the peer's copy of a shared variable, in the cluster block of rank `rank`
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
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// NV vectors of 16 bytes a thread and round
template <int NV, bool HALF>
__global__ void __launch_bounds__(T, NV <= 4 ? 4 : 2) logprobs_kernel(const Args a) {
  pdl_begin();
  constexpr int VW = HALF ? 8 : 4;
  constexpr float LOG2E = 1.4426950408889634f;
  __shared__ Smem sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int row = blockIdx.x / ranks;
  using E = typename std::conditional<HALF, __half, float>::type;
  const E *x = reinterpret_cast<const E *>(a.x) + (int64_t)row * a.stride;
  // whole vectors from the first 16-byte boundary on; the few values before and behind them are the first block's
  const int lead = min(a.n, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(E)));
  const int vecs = (a.n - lead) / VW, tail = lead + vecs * VW;
  const int per = (vecs + (int)ranks - 1) / (int)ranks;
  const int v0 = min(vecs, (int)rank * per), v1 = min(vecs, v0 + per);
  const uint4 *xv = reinterpret_cast<const uint4 *>(x + lead);

  float m = -INFINITY, S = 0.0f, Tm = 0.0f;  // of this thread's values so far, relative to m (the block's)
  int have = 0;                              // entries of sm.best
  const int rounds = max(1, (v1 - v0 + T * NV - 1) / (T * NV));
  for (int round = 0; round < rounds; round++) {
    const int base = v0 + round * T * NV + tid;
    uint4 u[NV];
    int mine = 0;  // vectors of this thread
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (base + i * T < v1) {
        u[i] = __ldcs(xv + base + i * T);
        mine = i + 1;
      }
    float edge = -INFINITY;  // the odd value of this thread
    int edge_id = -1;
    if (rank == 0 && round == 0) {
      if (tid < lead) edge_id = tid;
      else if (tid >= 32 && tail + tid - 32 < a.n) edge_id = tail + tid - 32;
      if (edge_id >= 0) edge = (float)x[edge_id];
    }
    auto unpacked = [&](int i, float (&y)[VW]) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (HALF) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
          y[(2 * j) % VW] = f.x, y[(2 * j + 1) % VW] = f.y;
        } else {
          y[j % VW] = __uint_as_float(w[j]);
        }
      }
    };
    float big = edge;
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (i < mine) {
        float y[VW];
        unpacked(i, y);
#pragma unroll
        for (int j = 0; j < VW; j++) big = max_nan(big, y[j]);
      }
    const float m_new = max_nan(m, block_max(big, sm.part[0]));
    if (m_new != m) {  // (NaN too: every sum is NaN from here on)
      const float by = m == -INFINITY ? 0.0f : ex2((m - m_new) * LOG2E);
      Tm = by == 0.0f ? 0.0f : (Tm + S * (m - m_new)) * by;
      S *= by;
      m = m_new;
    }
    // e = 2^((x - m) log2 e); x - m is held above -1e4, where e is 0 and e (x - m) too
    auto add = [&](float y) {
      const float d = fmaxf(y - m, -1e4f), e = ex2(d * LOG2E);
      S += e;
      Tm = __fmaf_rn(e, d, Tm);
    };
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (i < mine) {
        float y[VW];
        unpacked(i, y);
#pragma unroll
        for (int j = 0; j < VW; j++) add(y[j]);
      }
    if (edge_id >= 0) add(edge);

    if (a.k == 0) continue;
    // ---- the best k of this round and the rounds before
    uint32_t key = mine > 0 || edge_id >= 0 ? key_of(big) : 0;
    {
      // the ceil(k / 8)-th largest of the warp's thread maxima
      uint32_t rest = key, low = 0;
      for (int j = (a.k + WARPS - 1) / WARPS; j > 0; j--) {
        low = __reduce_max_sync(0xffffffffu, rest);
        const uint32_t holds = __ballot_sync(0xffffffffu, rest == low);
        if (lane == __ffs(holds) - 1) rest = 0;
      }
      if (lane == 0) sm.low[warp] = low;
      if (tid == 0) sm.count = 0;
    }
    __syncthreads();
    uint32_t low = sm.low[0];
#pragma unroll
    for (int w = 1; w < WARPS; w++) low = min(low, sm.low[w]);
    if (have == a.k) low = max(low, (uint32_t)(sm.best[a.k - 1] >> 32));
    auto each = [&](auto &&f) {
      if (key >= low && key) {
#pragma unroll
        for (int i = 0; i < NV; i++)
          if (i < mine) {
            float y[VW];
            unpacked(i, y);
            const int id = lead + (base + i * T) * VW;
#pragma unroll
            for (int j = 0; j < VW; j++) f(key_of(y[j]), id + j);
          }
        if (edge_id >= 0) f(key_of(edge), edge_id);
      }
    };
    each([&](uint32_t q, int id) {
      if (q >= low) {
        const int at = atomicAdd(&sm.count, 1);
        if (at < LIST) sm.list[at] = entry_of(q, id);
      }
    });
    __syncthreads();
    int listed = sm.count;
    if (listed > LIST - K_MOST) {
      // one after the other: the largest below the one picked last
      uint64_t last = ~0ull;
      listed = 0;
      for (; listed < a.k; listed++) {
        uint64_t pick = 0;
        each([&](uint32_t q, int id) {
          const uint64_t e = entry_of(q, id);
          if (e < last && e > pick) pick = e;
        });
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
      __syncthreads();
    }
    if (tid < have) sm.list[listed + tid] = sm.best[tid];
    listed += have;
    __syncthreads();
    for (int i = tid; i < listed; i += T) {
      const uint64_t e = sm.list[i];
      int better = 0;
      for (int j = 0; j < listed; j++) better += sm.list[j] > e;
      if (better < a.k) sm.best[better] = e;
    }
    have = min(a.k, listed);
    __syncthreads();
  }

  // ---- the block's sums, then the cluster's in the first block
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    S += __shfl_xor_sync(0xffffffffu, S, d);
    Tm += __shfl_xor_sync(0xffffffffu, Tm, d);
  }
  if (lane == 0) sm.part[1][warp] = S, sm.part[2][warp] = Tm;
  if (tid >= have && tid < a.k) sm.best[tid] = 0;
  __syncthreads();
  if (tid == 0) {
    S = Tm = 0.0f;
    for (int w = 0; w < WARPS; w++) S += sm.part[1][w], Tm += sm.part[2][w];
    sm.mst[0] = m, sm.mst[1] = S, sm.mst[2] = Tm;
  }
  if (ranks > 1) cluster_sync();
  else __syncthreads();
  if (rank != 0) {
    cluster_sync();  // the first block reads this one's shared memory until then
    return;
  }
  float M = -INFINITY, sum = 0.0f, dot = 0.0f;
  {
    float pm[8], ps[8], pt[8];
#pragma unroll
    for (int r = 0; r < 8; r++)
      if (r < (int)ranks) pm[r] = peer(&sm.mst[0], r), ps[r] = peer(&sm.mst[1], r), pt[r] = peer(&sm.mst[2], r);
    if (tid < (int)ranks * a.k) sm.all[tid] = peer(&sm.best[tid % a.k], tid / a.k);
#pragma unroll
    for (int r = 0; r < 8; r++)
      if (r < (int)ranks) M = max_nan(M, pm[r]);
#pragma unroll
    for (int r = 0; r < 8; r++)
      if (r < (int)ranks && pm[r] != -INFINITY) {
        const float d = pm[r] - M, by = ex2(d * LOG2E);
        sum += ps[r] * by;
        if (by != 0.0f) dot += (pt[r] + ps[r] * d) * by;
      }
  }
  if (ranks > 1) cluster_sync();
  else __syncthreads();
  // no finite largest logit (all masked, an infinity, a NaN): no distribution
  const bool fine = fabsf(M) < INFINITY;
  const float logS = fine ? logf(sum) : __uint_as_float(0x7fffffffu);
  if (tid == 0) {
    if (a.logprob) {
      const int t = a.targets[row];
      a.logprob[row] = t >= 0 && t < a.n ? ((float)x[t] - M) - logS : __uint_as_float(0x7fffffffu);
    }
    if (a.entropy) a.entropy[row] = logS - __fdiv_rn(dot, sum);
  }
  if (!fine) {
    if (tid < a.k) {
      a.ids[(int64_t)row * a.k + tid] = -1;
      a.top[(int64_t)row * a.k + tid] = logS;
    }
  } else if (tid < (int)ranks * a.k) {
    // the place of each block's entries among all of them
    const uint64_t e = sm.all[tid];
    int better = 0;
    for (int j = 0; j < (int)ranks * a.k; j++) better += sm.all[j] > e;
    if (e && better < a.k) {
      const int64_t at = (int64_t)row * a.k + better;
      a.ids[at] = ~(int)(uint32_t)e;
      a.top[at] = (value_of((uint32_t)(e >> 32)) - M) - logS;
    }
  }
}

template <bool HALF>
int launch_logprobs(const Args &a, int count, cudaStream_t stream) {
  constexpr int VW = HALF ? 8 : 4, FEW = 16 / VW, MANY = 64 / VW;
  // blocks of a row: enough for its values to stay in registers, more while the GPU has room for all rows' blocks
  const int vecs = (a.n + VW - 1) / VW;
  int ranks = 1;
  while (ranks < 8 && (vecs > ranks * T * MANY || (count * ranks * 2 <= 148 && vecs > ranks * T))) ranks *= 2;
  const bool few = (vecs + ranks - 1) / ranks <= T * FEW;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)count * ranks);
  cfg.blockDim = dim3(T);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_on() ? 2 : 1;
  (void)cudaLaunchKernelEx(&cfg, few ? logprobs_kernel<FEW, HALF> : logprobs_kernel<MANY, HALF>, a);
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
    const Args a = {logprob, entropy, top_logprob, top_id, logits, targets, stride, n, k};
    return half ? launch_logprobs<true>(a, count, as_stream(stream)) : launch_logprobs<false>(a, count, as_stream(stream));
  } catch (...) {
    return fail(B200FWD_EINVAL, "logprobs: exception");
  }
}
