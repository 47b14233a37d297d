// cache8_attention_tc.cu — attention over the paged 8-bit cache for blocks of tokens (requests of more than ROWS_FEW
// query rows a kv head), on the 5th-generation tensor cores: the numbers of cache8_attention.cu, whose comment has the
// mathematics (float16 pairs for float32, scales outside the products, weights relative to the largest term).
//
// A thread block takes 256 (float16) or 128 (float32) rows of one request and kv head, in tiles of 128 (row x: query head
// x % group of the request's token x / group, so the heads that share a kv head share its keys), and walks their
// positions in steps of 64. 640 threads (float32 with heads of up to 64: warps 0..3 bring the cache, and warps 4..7 and 8..11
// are the softmax of even and of odd steps, each with a running maximum and sum of its own):
//   warps 0..7 bring the cache: int8 keys and values by 16-byte loads one step ahead, widened to float16 (exact) into
//     shared memory in the tensor cores' 128-byte swizzled layout; a step's four units' scales beside them. Positions
//     are rows of both: for K Q^T they run along N, for P V along K, and the values' operand is described as major along
//     the head, so nothing is transposed;
//   warps 8..11 the softmax of the first tile, a thread a row (TMEM lane): scores from TMEM, weights as float16 (float32
//     queries: a high and a low part, in the two halves of the scores' columns) back over them;
//   warps 12..15, float16: the softmax of the second tile. The products add up in TMEM, which is rescaled there when a
//     row's maximum moves. float32: they add up each step's product in registers. (The tensor cores' float32 sums are
//     cut off rather than rounded: over 2048 positions that came to 2.5e-6 of the outputs, of one step it is nothing.)
//   warps 16..19 issue the products, two a tile: S = Q K^T (M 128, N 64; float32: once for each part of Q) and O = P V
//     (M 128, N head size; float32: once for each part of P) with P read from TMEM.
// What bounds it, in cycles. Float16, heads of 128: a step of both tiles takes 2330, of which the products are 1540 (S with
// its N of 64 at half rate: 63 for each 16 of K, as Q comes from shared memory every time; P V 66), exponentials 1024,
// issue slots 1400; a block begins and ends in 15,000 (the queries, the first keys, the first scores; rows out) beside 30
// steps on average. Float32, heads of 64: 1550 a step of one tile (one warpgroup of softmax: 2060), of which the products
// are about 900; each softmax step takes 2300 to 2600, twice its instructions' issue slots.
// Measured: 8 requests that add 260 to 509 tokens to contexts of up to 4500, 32 query and 8 kv heads of 128, float16: 168 us
// (0.66 PFLOP/s of what the masks leave); 4 whole prompts of 2048 tokens, 8 heads of 64, float32: 90 us.
// TMEM (512 columns), float16: tile t's two score buffers at 128 t + {0, 64}, its O at 256 + t * head size; float32: three
// score buffers (heads of up to 64: four) at 64 u, two of O behind them.
// Every wait is bounded: past it the kernel sets the scratch's error word (b200k_cache8_attention_check) and runs to its end.
#include <string>

#include "cache8_attention.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace cache8 {
namespace {

using namespace tc;

constexpr int QT = 128, KT = 64, THREADS = 640, KU = KT / UNIT;
// Requests that are taken in order of their lengths. Measured, sorted and not (prompt blocks over up to 4000 positions, 32 query
// and 8 kv heads of 128, float16): 8 requests 121 and 127 us, 64 176 and 216; 65, with a limit of 512, 181 and 217, 128 362
// and 385.
constexpr int SORTED = 64;

template <int HP, bool HALF>
struct Tc {
  static constexpr int TILES = HALF ? 2 : 1;
  static constexpr int CHUNKS = HP / 64;  // 128-byte columns of 64 float16
  static constexpr int PARTS = HALF ? 1 : 2;
  static constexpr int STAGES = 4;
  // float32, heads of up to 64: two warpgroups of softmax (of even and odd steps), and four warps that bring the cache
  static constexpr int SOFT = !HALF && HP == 64 ? 2 : 1, BRINGERS = SOFT == 2 ? 128 : 256;
  static constexpr int SBUF = HALF ? 2 : 2 + SOFT;  // score buffers of a tile
  struct Smem {
    alignas(1024) uint8_t q[TILES][PARTS][CHUNKS][QT * 128];
    alignas(1024) uint8_t k[STAGES][CHUNKS][KT * 128];
    alignas(1024) uint8_t v[STAGES][CHUNKS][KT * 128];
    alignas(16) float4 sc[STAGES][KU];  // a unit's {key scale, log2(value scale), 1 / value scale}
    // float32: the maxima that a step's weights are relative to (softmax is up to SBUF + 1 steps ahead of the sums); at the
    // end each warpgroup's sums and maxima; the powers of two that the queries were divided by
    float ref[8][QT], l[SOFT][QT], m[SOFT][QT], power[QT];
    uint64_t q_full, kv_full[STAGES], kv_empty[STAGES];
    uint64_t s_full[TILES][SBUF], p_full[TILES][SBUF], pv_done[TILES][SBUF], o_free[2], ref_full[8], l_full, mma_done;
    uint32_t tmem_base;
    int part[2][THREADS / 32], found[2];
    int2 of[SORTED];                    // the requests' positions and groups of tiles
    int2 row[TILES][QT];                // a row's token (of all; -1: there is none) and query head
  };
};

// Waits for the phase of `parity`; false when that took 2 s, or another wait did (the error word is set then). Without a
// suspend-time hint: from a thread of a warp's to another's and back takes 281 cycles so, with a hint of 1 ms 671.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, int *error, int code) {
  const uint32_t addr = smem_u32(bar);
  uint64_t begun = 0, now;
  for (uint32_t i = 1;; i++) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 255) == 0) {
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
      if (begun == 0) begun = now;
      if (*(volatile int *)error) return false;
      if (now - begun > 2000000000ull) {
        atomicCAS(error, 0, code);
        return false;
      }
    }
  }
}
// The thread of a converged warp that issues its products. (elect.sync rather than a lane's number: the products' operands
// go through the warp's uniform registers, and what the compiler makes of a branch on the lane, predicates among it, left
// other lanes' values in them; with a predicate of one's own on every product a product took 100 cycles to issue, 66 so.)
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p;
}
// D (+)= A B, A from shared memory or from TMEM (float16 pairs along K), B from shared memory
template <bool ADD>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "n"(ADD ? 1 : 0)
      : "memory");
}
template <bool ADD>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "n"(ADD ? 1 : 0)
      : "memory");
}
// The values: 128-byte rows of 64 head values, a row a position, swizzled. Major along the head (N): the next 64 of the
// head `chunk` bytes on, the next 8 positions (K) 1024.
__device__ __forceinline__ uint64_t desc_head_major(const void *p, uint32_t chunk) {
  uint64_t d = 0;
  d |= (smem_u32(p) >> 4) & 0x3fff;
  d |= (uint64_t)(chunk >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
constexpr uint32_t B_MAJOR_N = 1u << 16;

// 32 TMEM columns of this thread's lane, not waited for
__device__ __forceinline__ void ld32(uint32_t taddr, float *r) {
  uint32_t *u = reinterpret_cast<uint32_t *>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr));
}
__device__ __forceinline__ void st8(uint32_t taddr, const uint32_t *u) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(u[0]),
               "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}
// every load of this thread has arrived; x: what they were into (so that nothing reads it earlier)
__device__ __forceinline__ void wait_ld32(float *x) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7]), "+f"(x[8]),
                 "+f"(x[9]), "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]), "+f"(x[14]), "+f"(x[15]), "+f"(x[16]),
                 "+f"(x[17]), "+f"(x[18]), "+f"(x[19]), "+f"(x[20]), "+f"(x[21]), "+f"(x[22]), "+f"(x[23]), "+f"(x[24]),
                 "+f"(x[25]), "+f"(x[26]), "+f"(x[27]), "+f"(x[28]), "+f"(x[29]), "+f"(x[30]), "+f"(x[31])
               :
               : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float reciprocal(float x) {  // within 1 of the last place
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// One step of this thread's row: 64 scores from tS, their weights over them. EDGE: some of the tile's rows don't see all
// of the step; limit: the last position that this row sees, from the step's first. qf: what a score takes besides its key
// scale, log2(e) / sqrt(hs) and the power of two that the row was divided by. m, l: the row's running maximum and sum.
// The weights are relative to m, float32's to the step's own maximum (its products are added to the sums one step at a
// time, so a step far below the others keeps its bits). settle(ref, by): called by the whole warp once that is known: ref,
// and, float16, what the row's sums go down by where some row's m moved, else -1. (The next step's scores, loaded while
// this one's last weights are worked out, cost more than they saved: 189 us for 172, 102 for 97.)
template <int HP, bool HALF, bool EDGE, typename Settle>
__device__ __forceinline__ void softmax_step(uint32_t tS, const float4 *sc, float qf, int limit, float &m, float &l,
                                             Settle &&settle) {
  float x[KT];
  ld32(tS, x);
  ld32(tS + 32, x + 32);
  float c[KU], lg[KU], inv[KU];
#pragma unroll
  for (int u = 0; u < KU; u++) {
    const float4 s = sc[u];
    c[u] = s.x * qf, lg[u] = s.y, inv[u] = s.z;
    // (a unit that the row does not see may have any scales, NaN too)
    if (EDGE && u * UNIT > limit) c[u] = 1.0f, lg[u] = 0.0f, inv[u] = 0.0f;
    // (a factor of 0, of a row or keys of zeros, as the least, which moves no exponent: 0 times a masked -inf is no number)
    if (EDGE && c[u] < 1e-30f) c[u] = 1e-30f;
  }
  wait_ld32(x);
  wait_ld32(x + 32);
  float most = -INFINITY;
#pragma unroll
  for (int u = 0; u < KU; u++) {
    if (EDGE) {
#pragma unroll
      for (int i = 0; i < UNIT; i++)
        if (u * UNIT + i > limit) x[u * UNIT + i] = -INFINITY;
    }
    float top = x[u * UNIT];
#pragma unroll
    for (int i = 1; i + 1 < UNIT; i += 2) top = max3(top, x[u * UNIT + i], x[u * UNIT + i + 1]);
    top = fmaxf(top, x[u * UNIT + UNIT - 1]);
    most = fmaxf(most, __fmaf_rn(top, c[u], lg[u]));
  }
  float ref = most, step_by = 1.0f, step_l = 0.0f;
  if (!HALF) {
    const float top = fmaxf(m, most);
    l *= m == top ? 1.0f : ex2(m - top);
    step_by = most == top ? 1.0f : ex2(most - top);
    m = top;
    settle(most, -1.0f);
  } else {
    if (__any_sync(0xffffffffu, most > m + RESCALE)) {
      const float top = fmaxf(m, most), by = m == top ? 1.0f : ex2(m - top);
      l *= by, m = top;
      settle(m, by);
    } else {
      settle(m, -1.0f);
    }
    ref = m;
  }
  const float from = ref == -INFINITY ? 0.0f : ref - LIFT;
#pragma unroll
  for (int u = 0; u < KU; u++) {
    const uint64_t c2 = f2(c[u], c[u]), a2 = f2(lg[u] - from, lg[u] - from);
    uint64_t sum = f2(0.0f, 0.0f);
    uint32_t hi[UNIT / 2], lo[UNIT / 2];
#pragma unroll
    for (int i = 0; i < UNIT; i += 2) {
      const uint64_t e = fma_2(f2(x[u * UNIT + i], x[u * UNIT + i + 1]), c2, a2);
      const float w0 = ex2(lo_of(e)), w1 = ex2(hi_of(e));
      sum = add_2(sum, f2(w0, w1));
      hi[i / 2] = pack(w0, w1);
      if (!HALF) {
        const float2 b = unpack(hi[i / 2]);
        lo[i / 2] = pack(w0 - b.x, w1 - b.y);
      }
    }
    (HALF ? l : step_l) = __fmaf_rn(lo_of(sum) + hi_of(sum), inv[u], HALF ? l : step_l);
    st8(tS + 8 * u, hi);
    if (!HALF) st8(tS + 32 + 8 * u, lo);
  }
  if (!HALF) l = __fmaf_rn(step_l, step_by, l);
  wait_st();
}

template <int HP, bool HALF>
__global__ void __launch_bounds__(THREADS, 1) cache8_attention_tc_kernel(const Args a) {
  using S = Tc<HP, HALF>;
  constexpr int STAGES = S::STAGES, PARTS = S::PARTS, TILES = S::TILES, SBUF = S::SBUF, SOFT = S::SOFT, BRINGERS = S::BRINGERS;
  extern __shared__ uint8_t raw[];
  typename S::Smem &s = *reinterpret_cast<typename S::Smem *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  pdl_begin();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // (a tile group's heads side by side)
  const int h = blockIdx.x % a.nkv, index = blockIdx.x / a.nkv;
  int *error = &a.meta[-1].y;

  // ---- which request's which group of TILES tiles: a request's last rows, which see the most positions, first, and up to
  // SORTED requests the longest first (a block's time is its positions'; what starts last should be short)
  int total = 0, astray = 0;
  if (tid == 0) s.found[0] = -1;
  for (int base = 0; base < a.n_seqs; base += THREADS) {
    const int i = base + tid;
    int groups = 0;
    bool own = false;
    if (i < a.n_seqs) {
      const Request r = request_of(a, i);
      own = r.astray;
      groups = r.fresh * a.group > a.rows_most ? (r.fresh * a.group + TILES * QT - 1) / (TILES * QT) : 0;
      if (a.n_seqs <= SORTED) s.of[tid] = make_int2(r.length, groups);
    }
    int upto = groups;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    own = __any_sync(0xffffffffu, own);
    __syncthreads();
    if (lane == 31) s.part[0][warp] = upto, s.part[1][warp] = own;
    __syncthreads();
    int before = total;
    for (int w = 0; w < min(THREADS / 32, (a.n_seqs - base + 31) / 32); w++) {
      if (w < warp) before += s.part[0][w];
      total += s.part[0][w];
      astray |= s.part[1][w];
    }
    before += upto - groups;
    if (a.n_seqs <= SORTED && i < a.n_seqs) {
      before = 0;
      const int length = s.of[tid].x;
      for (int k = 0; k < a.n_seqs; k++) {
        const int2 o = s.of[k];
        if (o.x > length || (o.x == length && k < i)) before += o.y;
      }
    }
    const int x = index - before;
    if (x >= 0 && x < groups) s.found[0] = i, s.found[1] = groups - 1 - x;
  }
  if (astray) return;  // starts that don't ascend
  __syncthreads();
  const int req = s.found[0];
  if (req < 0) return;
  const Request r = request_of(a, req);
  const int rows = r.fresh * a.group, cap = a.width * a.block, row0 = s.found[1] * TILES * QT;
  // steps of each tile: up to its last row's position (and within the table's row)
  int steps[2] = {0, 0}, most_steps = 0;
#pragma unroll
  for (int t = 0; t < TILES; t++) {
    const int x = min(rows, row0 + (t + 1) * QT) - 1;  // the tile's last row
    const int seen = x < row0 + t * QT ? 0 : min(r.length - r.fresh + x / a.group + 1, cap);
    steps[t] = max(0, (seen + KT - 1) / KT);
    most_steps = max(most_steps, steps[t]);
  }

  if (tid == 0) {
    mbar_init(&s.q_full, TILES * SOFT * QT);
    for (int i = 0; i < STAGES; i++) {
      mbar_init(&s.kv_full[i], BRINGERS);
      mbar_init(&s.kv_empty[i], TILES);
    }
    for (int t = 0; t < TILES; t++) {
      for (int u = 0; u < SBUF; u++) {
        mbar_init(&s.s_full[t][u], 1);
        mbar_init(&s.p_full[t][u], 4);
        mbar_init(&s.pv_done[t][u], 1);
      }
    }
    for (int u = 0; u < 2; u++) mbar_init(&s.o_free[u], 4);
    for (int u = 0; u < 8; u++) mbar_init(&s.ref_full[u], 4);
    mbar_init(&s.l_full, 4 * SOFT);
    mbar_init(&s.mma_done, 2 * TILES);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem_base)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s.tmem_base;
  auto tS = [&](int t, int u) { return tmem + (uint32_t)((t * SBUF + u) * KT); };
  auto tO = [&](int t) { return tmem + (uint32_t)((TILES * SBUF) * KT + t * HP); };  // float32: t the buffer

  // this thread's row of its tile (softmax and summing threads; TMEM lane y)
  const int y = tid & 127, t_own = HALF && warp >= 12 ? 1 : 0, x_own = row0 + t_own * QT + y;
  const bool on = x_own < rows;
  const int token = on ? x_own / a.group : 0, head = h * a.group + (on ? x_own % a.group : 0);
  const int pos = on ? r.length - r.fresh + token : -1;
  const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
  // Output rows go through the tile's queries' place in shared memory, so that a warp writes whole rows: 8 values z of
  // this thread's row from value d on, then all the warp's rows
  constexpr int PIECES = HP * (HALF ? 2 : 4) / 16;
  auto put = [&](int d, const float (&z)[8]) {
    uint8_t *row = &s.q[t_own][0][0][0] + y * (PIECES * 16);
    if (HALF) {
      *reinterpret_cast<uint4 *>(row + (((d >> 3) ^ (y & 7)) << 4)) =
          make_uint4(pack(z[0], z[1]), pack(z[2], z[3]), pack(z[4], z[5]), pack(z[6], z[7]));
    } else {
      *reinterpret_cast<float4 *>(row + (((d >> 2) ^ (y & 7)) << 4)) = make_float4(z[0], z[1], z[2], z[3]);
      *reinterpret_cast<float4 *>(row + (((d >> 2) + 1 ^ (y & 7)) << 4)) = make_float4(z[4], z[5], z[6], z[7]);
    }
  };
  auto write = [&]() {
    constexpr int ES = HALF ? 2 : 4;
    const int piece = lane % PIECES;
    s.row[t_own][y] = make_int2(on ? r.first + token : -1, head);
    __syncwarp();
#pragma unroll 1
    for (int i = lane / PIECES; i < 32; i += 4 * (32 / PIECES)) {
      uint4 z[4];
      int2 of[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int row = (y & ~31) + i + u * (32 / PIECES);
        of[u] = s.row[t_own][row];
        z[u] = *reinterpret_cast<const uint4 *>(&s.q[t_own][0][0][0] + (row * PIECES + (piece ^ (row & 7))) * 16);
      }
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (of[u].x >= 0 && piece * 16 < a.hs * ES)
          *reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(a.out) +
                                     (of[u].x * a.out_stride + (int64_t)of[u].y * a.hs) * ES + piece * 16) = z[u];
    }
  };
  // 1 / the row sum; a row that sees nothing is 0, one past its table's row, without any weight (all its scores -inf, of an
  // infinite query) or after a wait that gave up NaN
  auto inverse = [&](float l, bool ok) {
    return pos < 0 && ok ? 0.0f : !ok || pos >= cap || l == 0.0f ? __uint_as_float(0x7fffffffu) : __fdiv_rn(1.0f, l);
  };

  // (the launch's 640 x 96 registers: 128 x (64 + 64 + 144 + 168 + 40), SOFT 2 128 x (64 + 128 + 128 + 120 + 40), float16
  // 128 x (64 + 64 + 152 + 152 + 48))
  if (warp < BRINGERS / 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // ---- the cache: a thread brings 16 bytes of rows brow + i * PER (CH pieces a row) of keys and of values. Eight threads
    // in a row take four pieces of two rows, which go to eight different 16-byte columns of the swizzled lines.
    constexpr int CH = HP / 16, PER = BRINGERS / CH, R = KT / PER;
    const int32_t *table = a.tables + (int64_t)req * a.width;
    const int piece = (tid & 3) + (tid >> 3) % (CH / 4) * 4, brow = (tid >> 2 & 1) + (tid >> 3) / (CH / 4) * 2;
    const bool in_head = piece * 16 < a.hs;
    // table entries from held on are no row's to see (or NaN rows')
    const int held = min(a.width, (r.length + a.block - 1) / a.block);
    const int page_bytes = a.nkv * a.block * a.hs, head_bytes = h * a.block * a.hs + piece * 16;
    const int step_blocks = KT / a.block, step_rest = KT % a.block;
    // a row's place: its block in the table, its position in the block
    struct Place {
      int block, at;
    };
    auto place_of = [&](int p) { return Place{p / a.block, p % a.block}; };
    auto forward = [&](Place &p) {
      p.block += step_blocks, p.at += step_rest;
      if (p.at >= a.block) p.at -= a.block, p.block++;
    };
    auto page_of = [&](const Place &p) { return p.block < held ? table[p.block] : -1; };
    // (what is no block's, or past the head, stays any integers: the scales are NaN there, the queries 0)
    auto load = [&](uint4 &k, uint4 &v, int page, int at) {
      if ((uint32_t)page < (uint32_t)a.blocks && in_head) {
        const int64_t off = (int64_t)page * page_bytes + (head_bytes + at * a.hs);
        k = *reinterpret_cast<const uint4 *>(a.kc + off), v = *reinterpret_cast<const uint4 *>(a.vc + off);
      }
    };
    auto widened = [&](uint8_t *tile, int i, const uint4 &v) {
      const int row = brow + i * PER;
      uint8_t *dst = tile + (piece >> 2) * (KT * 128) + row * 128;
      const uint32_t w[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
      const int c0 = (piece & 3) * 2;
      *reinterpret_cast<uint4 *>(dst + ((c0 ^ (row & 7)) << 4)) =
          make_uint4(widen<0x4140>(w[0]), widen<0x4342>(w[0]), widen<0x4140>(w[1]), widen<0x4342>(w[1]));
      *reinterpret_cast<uint4 *>(dst + (((c0 + 1) ^ (row & 7)) << 4)) =
          make_uint4(widen<0x4140>(w[2]), widen<0x4342>(w[2]), widen<0x4140>(w[3]), widen<0x4342>(w[3]));
    };
    Place far[R];  // of the step after next
    int next[R], next_at[R];  // the next step's blocks and places in them
    uint4 k[R], v[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
      k[i] = v[i] = make_uint4(0, 0, 0, 0);
      far[i] = place_of(brow + i * PER);
      const int page = most_steps > 0 ? page_of(far[i]) : -1;
      load(k[i], v[i], page, far[i].at);
      forward(far[i]);
      next[i] = most_steps > 1 ? page_of(far[i]) : -1, next_at[i] = far[i].at;
      forward(far[i]);
    }
    // threads 0..3: a unit's scales, one step ahead, its block two
    Place sfar = place_of((tid & 3) * UNIT);
    int spage = -1;
    float ks = 0.0f, vs = 0.0f;
    auto scales = [&](int p) {
      const bool ok = (uint32_t)p < (uint32_t)a.blocks;
      ks = ok ? a.ks[(int64_t)p * a.nkv + h] : __uint_as_float(0x7fffffffu);
      vs = ok ? a.vs[(int64_t)p * a.nkv + h] : __uint_as_float(0x7fffffffu);
    };
    if (tid < KU && most_steps > 0) {
      scales(page_of(sfar));
      forward(sfar);
      spage = page_of(sfar);
      forward(sfar);
    }
    for (int j = 0; j < most_steps; j++) {
      const int slot = j % STAGES;
      if (!wait_for(&s.kv_empty[slot], ((j / STAGES) & 1) ^ 1, error, 101)) break;
      const bool more = j + 1 < most_steps;
#pragma unroll
      for (int i = 0; i < R; i++) {
        widened(s.k[slot][0], i, k[i]);
        widened(s.v[slot][0], i, v[i]);
        if (more) load(k[i], v[i], next[i], next_at[i]);
        next[i] = page_of(far[i]), next_at[i] = far[i].at;
        forward(far[i]);
      }
      if (tid < KU) {
        const float w = !(vs < LEAST) ? vs : LEAST;
        s.sc[slot][tid] = make_float4(ks, __log2f(w), reciprocal(w), 0.0f);
        if (more) {
          scales(spage);
          spage = page_of(sfar);
          forward(sfar);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&s.kv_full[slot]);
    }
  } else if (warp >= 16) {
    if (HALF) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // A warp each for the scores' products and for the values', of each tile, and one thread of it: what such a thread waits
    // for and works out between products takes a few hundred cycles, in which the others keep the tensor cores busy. What
    // it computes for a product is a sum: the operands' descriptors are the first ones', with a multiple of 16 bytes added
    // to the address in their low bits.
    const int t = (warp - 16) >> 1;
    if (t < TILES && elected()) {
      constexpr int PART = S::CHUNKS * QT * 128 / 16, STAGE = S::CHUNKS * KT * 128 / 16;
      bool ok = true;
      auto wait = [&](uint64_t *bar, uint32_t parity, int code) { ok = ok && wait_for(bar, parity, error, code); };
      if ((warp & 1) == 0) {
        const uint32_t id_s = idesc_f16(QT, KT);
        const uint64_t q0 = desc_sw128(s.q[t][0][0]), k0 = desc_sw128(s.k[0][0]);
        wait(&s.q_full, 0, 103);
        for (int j = 0; j < steps[t]; j++) {
          wait(&s.kv_full[j % STAGES], (j / STAGES) & 1, 104);
          wait(&s.pv_done[t][j % SBUF], ((j / SBUF) & 1) ^ 1, 107);  // the buffer's last weights have been used
          if (!ok) break;
          fence_after();
          const uint32_t d = tS(t, j % SBUF);
          const uint64_t kd = k0 + (j % STAGES) * STAGE;
          mma_ss<false>(d, q0, kd, id_s);
#pragma unroll
          for (int part = 0; part < PARTS; part++)
#pragma unroll
            for (int kk = 0; kk < HP / 16; kk++)
              if (part > 0 || kk > 0)
                mma_ss<true>(d, q0 + part * PART + (kk >> 2) * (QT * 8) + 2 * (kk & 3), kd + (kk >> 2) * (KT * 8) + 2 * (kk & 3),
                             id_s);
          mma_commit(&s.s_full[t][j % SBUF]);
        }
      } else {
        const uint32_t id_o = idesc_f16(QT, HP) | B_MAJOR_N;
        const uint64_t v0 = desc_head_major(s.v[0][0], KT * 128);
        for (int j = 0; j < most_steps; j++) {
          if (j >= steps[t]) {
            // the other tile's alone (an arrival a step, so not before the step is there)
            wait(&s.kv_full[j % STAGES], (j / STAGES) & 1, 108);
            if (!ok) break;
            mbar_arrive(&s.kv_empty[j % STAGES]);
            continue;
          }
          wait(&s.p_full[t][j % SBUF], (j / SBUF) & 1, 106);
          if (!HALF) wait(&s.o_free[j & 1], ((j >> 1) & 1) ^ 1, 105);
          if (!ok) break;
          fence_after();
          const uint32_t d = tO(HALF ? t : j & 1), p = tS(t, j % SBUF);
          const uint64_t vd = v0 + (j % STAGES) * STAGE;
          if (HALF && j > 0) mma_ts<true>(d, p, vd, id_o);
          else mma_ts<false>(d, p, vd, id_o);
#pragma unroll
          for (int part = 0; part < PARTS; part++)
#pragma unroll
            for (int kk = 0; kk < KT / 16; kk++)
              if (part > 0 || kk > 0) mma_ts<true>(d, p + 32 * part + 8 * kk, vd + 128 * kk, id_o);
          mma_commit(&s.pv_done[t][j % SBUF]);
          mma_commit(&s.kv_empty[j % STAGES]);  // (this step's scores came before its weights)
        }
      }
      mma_commit(&s.mma_done);
    }
    __syncwarp();
    // every product issued has completed before the block frees TMEM
    if (warp == 16) wait_for(&s.mma_done, 0, error, 114);
  } else if (!HALF && warp >= 12) {
    if (SOFT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    // ---- float32: the rows' sums, a step's product at a time
    const int n = steps[0];
    float acc[HP];
#pragma unroll
    for (int i = 0; i < HP; i++) acc[i] = 0.0f;
    float top = -INFINITY;
    bool ok = true;
    for (int j = 0; j < n && ok; j++) {
      ok = wait_for(&s.ref_full[j & 7], (j >> 3) & 1, error, 121);
      ok = wait_for(&s.pv_done[0][j % SBUF], (j / SBUF) & 1, error, 122) && ok;
      ok = __all_sync(0xffffffffu, ok);
      // both to the larger maximum
      const float ref = s.ref[j & 7][y], to = fmaxf(top, ref);
      const float old_by = top == to ? 1.0f : ex2(top - to), new_by = ref == to ? 1.0f : ex2(ref - to);
      const uint64_t old2 = f2(old_by, old_by), new2 = f2(new_by, new_by);
      top = to;
      fence_after();
#pragma unroll
      for (int ch = 0; ch < HP / 16; ch++) {
        uint32_t o[16];
        tmem_ld<16>(tO(j & 1) + lane_base + ch * 16, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const uint64_t z = fma_2(f2(acc[ch * 16 + i], acc[ch * 16 + i + 1]), old2,
                                   mul_2(f2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), new2));
          acc[ch * 16 + i] = lo_of(z), acc[ch * 16 + i + 1] = hi_of(z);
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.o_free[j & 1]);
    }
    ok = wait_for(&s.l_full, 0, error, 123) && ok;
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < SOFT; i++) l += s.l[i][y] * (s.m[i][y] == top ? 1.0f : ex2(s.m[i][y] - top));
    const float by = inverse(l, ok);
#pragma unroll
    for (int d = 0; d < HP; d += 8) {
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; e++) z[e] = by == 0.0f ? 0.0f : acc[d + e] * by;
      put(d, z);
    }
    write();
  } else {
    if (HALF) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
    else if (SOFT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    // ---- the softmax of tile t_own. Its queries first, as float16 (float32: in two parts, by a power of two to below 2^15,
    // so that the low part, which ends at 2^-24, reaches down to 2^-39 of the row's largest) in the swizzled layout
    const int t = t_own, soft = SOFT == 2 ? (warp - BRINGERS / 32) >> 2 : 0;
    float qf = a.scale;
    s.row[t][y] = make_int2(on ? r.first + token : -1, head);  // (SOFT 2: both warpgroups write, the same)
    asm volatile("bar.sync %0, 128;" ::"r"(1 + t + soft) : "memory");
    {
      // a row by LANES threads, 8 values each; ROWS rows' loads in flight
      constexpr int LANES = HP / 8, AT_ONCE = 128 / LANES, ROWS = HALF ? 8 : 4;
      const int col = y % LANES * 8, sub = y / LANES;
#pragma unroll 1
      for (int first = sub + soft * (QT / SOFT); first < (soft + 1) * (QT / SOFT); first += ROWS * AT_ONCE) {
        uint4 raw[ROWS][HALF ? 1 : 2];
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
          const int2 of = s.row[t][first + i * AT_ONCE];
          const int64_t off = of.x * a.q_stride + (int64_t)of.y * a.hs + col;
          const uint4 *src = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(a.q) + off * (HALF ? 2 : 4));
          const bool in = of.x >= 0 && col < a.hs;  // (zeros past the head, as the keys have there)
#pragma unroll
          for (int e = 0; e < (HALF ? 1 : 2); e++) raw[i][e] = in ? src[e] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
          const int row = first + i * AT_ONCE;
          uint4 hi = raw[i][0], lo = hi;
          if (!HALF) {
            const uint4 w = raw[i][PARTS - 1];
            float z[8] = {__uint_as_float(hi.x), __uint_as_float(hi.y), __uint_as_float(hi.z), __uint_as_float(hi.w),
                          __uint_as_float(w.x),  __uint_as_float(w.y),  __uint_as_float(w.z),  __uint_as_float(w.w)};
            float top = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(z[k]));
#pragma unroll
            for (int d = LANES / 2; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            // (rows below 2^-112 as if they were of that size: the powers have to be whole float32)
            const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -112), 127) - 14;
            const float f = __uint_as_float((uint32_t)(127 - e) << 23);
            if (col == 0) s.power[row] = __uint_as_float((uint32_t)(127 + e) << 23);
            uint32_t p[4], q[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
              z[2 * k] *= f, z[2 * k + 1] *= f;
              p[k] = pack(z[2 * k], z[2 * k + 1]);
              const float2 b = unpack(p[k]);
              q[k] = pack(z[2 * k] - b.x, z[2 * k + 1] - b.y);
            }
            hi = make_uint4(p[0], p[1], p[2], p[3]), lo = make_uint4(q[0], q[1], q[2], q[3]);
          }
          const int at = row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4);
          *reinterpret_cast<uint4 *>(&s.q[t][0][col >> 6][at]) = hi;
          if (!HALF) *reinterpret_cast<uint4 *>(&s.q[t][PARTS - 1][col >> 6][at]) = lo;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&s.q_full);
      if (!HALF) {
        asm volatile("bar.sync 3, %0;" ::"n"(128 * SOFT) : "memory");
        qf = s.power[y] * a.scale;
      }
    }
    const int first_pos = r.length - r.fresh + (row0 + t * QT) / a.group;  // the tile's first row's
    const uint32_t o_col = tO(t) + lane_base;
    float m = -INFINITY, l = 0.0f;
    const int n = steps[t];
    bool ok = true;
    for (int j = soft; j < n && ok; j += SOFT) {
      // (the step's scales are there with its scores: the keys were complete before the scores were begun)
      ok = wait_for(&s.s_full[t][j % SBUF], (j / SBUF) & 1, error, 116);
      ok = wait_for(&s.kv_full[j % STAGES], (j / STAGES) & 1, error, 117) && ok;
      ok = __all_sync(0xffffffffu, ok);
      fence_after();
      auto settle = [&](float ref, float by) {
        if (!HALF) {
          s.ref[j & 7][y] = ref;
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.ref_full[j & 7]);
        } else if (by >= 0.0f && j > 0) {  // (whole warps come here: TMEM is read and written by whole warps)
          // O holds the steps so far: it goes to the new maxima once the last P V is done
          // (given up: O stays as it is, and the rows come out NaN)
          ok = __all_sync(0xffffffffu, wait_for(&s.pv_done[t][(j - 1) & 1], ((j - 1) >> 1) & 1, error, 109)) && ok;
          if (!ok) return;
          fence_after();
#pragma unroll
          for (int ch = 0; ch < HP / 16; ch++) {
            uint32_t o[16];
            tmem_ld<16>(o_col + ch * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
            st8(o_col + ch * 16, o);
            st8(o_col + ch * 16 + 8, o + 8);
          }
        }
      };
      // (rows that don't exist have pos -1: nothing of a step is theirs, and nothing of theirs is written)
      const uint32_t from = tS(t, j % SBUF) + lane_base;
      const float4 *sc = s.sc[j % STAGES];
      if (j * KT + KT - 1 > first_pos) softmax_step<HP, HALF, true>(from, sc, qf, pos - j * KT, m, l, settle);
      else softmax_step<HP, HALF, false>(from, sc, qf, 0, m, l, settle);
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.p_full[t][j % SBUF]);
    }
    if (!HALF) {
      s.l[soft][y] = ok ? l : __uint_as_float(0x7fffffffu), s.m[soft][y] = m;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.l_full);
    } else {
      if (n > 0) {
        ok = wait_for(&s.pv_done[t][(n - 1) & 1], ((n - 1) >> 1) & 1, error, 118) && ok;
        __syncwarp();
        fence_after();
      } else {
        ok = wait_for(&s.q_full, 0, error, 119) && ok;  // (the rows go where other warps still put queries)
      }
      const float by = inverse(l, ok);
      __syncwarp();
#pragma unroll 1
      for (int ch = 0; ch < HP / 32; ch++) {
        float o[32];
        if (n > 0) {
          ld32(o_col + ch * 32, o);
          wait_ld32(o);
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float z[8];
#pragma unroll
          for (int e = 0; e < 8; e++) z[e] = n > 0 && by != 0.0f ? o[i + e] * by : by;
          put(ch * 32 + i, z);
        }
      }
      write();
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 16) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int HP, bool HALF>
int launch_tc(const Args &a, cudaStream_t stream) {
  using S = Tc<HP, HALF>;
  auto kernel = cache8_attention_tc_kernel<HP, HALF>;
  const size_t smem = sizeof(typename S::Smem) + 1024;
  B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  // groups of tiles: all rows', and one more for every request that has any (at least rows_most + 1 rows each)
  const int64_t rows = (int64_t)a.n * a.group, requests = rows / (a.rows_most + 1);
  const int64_t groups = rows / (S::TILES * QT) + (requests < a.n_seqs ? requests : a.n_seqs);
  if (groups < 1) return 0;
  launch(kernel, dim3((unsigned)(groups * a.nkv)), dim3(THREADS), smem, stream, a);
  B200_LAUNCHED("cache8_attention_tc");
  return 0;
}

}  // namespace

int launch_attention8_prompts(const Args &a, bool half, cudaStream_t stream) {
  if (a.hs <= 64) return half ? launch_tc<64, true>(a, stream) : launch_tc<64, false>(a, stream);
  return half ? launch_tc<128, true>(a, stream) : launch_tc<128, false>(a, stream);
}

}  // namespace cache8
}  // namespace b200
