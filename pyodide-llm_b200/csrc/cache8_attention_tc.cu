// cache8_attention_tc.cu — attention over the paged 8-bit cache for blocks of tokens (requests of more than ROWS_FEW
// query rows a kv head), on the 5th-generation tensor cores: the numbers of cache8_attention.cu, whose comment has the
// mathematics (float16 pairs for float32, scales outside the products, weights relative to the largest term).
//
// A thread block takes two neighbouring tiles of 128 rows of one request and kv head (row x: query head x % group of the
// request's token x / group, so the heads that share a kv head share its keys) and walks their positions in steps of 64.
// 512 threads:
//   warps 0..3 bring the cache: int8 keys and values by 16-byte loads one step ahead, widened to float16 (exact) into
//     shared memory in the tensor cores' 128-byte swizzled layout, for both tiles at once; a step's four units'
//     scales beside them. Positions are rows of both: for K Q^T they run along N, for P V along K, and the values'
//     operand is described as major along the head, so nothing is transposed;
//   warps 4..7 and 8..11 the softmax of each tile, a thread a row (TMEM lane): scores from TMEM, weights as float16
//     (float32 queries: a high and a low part, in the two halves of the scores' columns) back over them;
//   warp 12 issues the products: S = Q K^T (M 128, N 64; float32: once for each part of Q) into one of a tile's two
//     score buffers, O += P V (M 128, N head size; float32: once for each part of P) with P read from TMEM.
// Bound by the tensor cores and the exponentials about alike (float16 queries, heads of 128: a step of two tiles is
// 1024 cycles of each), with the widening under both; float32 queries double the products.
// TMEM (512 columns): tile t's score buffers at 128 t + {0, 64}, its O at 256 + 128 t (64 t at heads of 64).
// Every wait is bounded: past it the kernel sets the scratch's error word and runs to its end.
#include <string>

#include "cache8_attention.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace cache8 {
namespace {

using namespace tc;

constexpr int QT = 128, KT = 64, THREADS = 512, KU = KT / UNIT;

template <int HP, bool HALF>
struct Tc {
  static constexpr int CHUNKS = HP / 64;              // 128-byte columns of 64 float16
  static constexpr int PARTS = HALF ? 1 : 2;          // of a float32 number
  static constexpr int STAGES = HP == 128 && !HALF ? 3 : 4;
  struct Smem {
    alignas(1024) uint8_t q[2][PARTS][CHUNKS][QT * 128];
    alignas(1024) uint8_t k[STAGES][CHUNKS][KT * 128];
    alignas(1024) uint8_t v[STAGES][CHUNKS][KT * 128];
    alignas(16) float4 sc[STAGES][KU];  // a unit's {key scale * log2(e) / sqrt(hs), log2(value scale), 1 / value scale}
    uint64_t q_full, kv_full[STAGES], kv_empty[STAGES];
    uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], mma_done;  // [tile][buffer]
    uint32_t tmem_base;
    int part[2][THREADS / 32], found[2];
  };
};

// A from TMEM (float16 pairs along K), B from shared memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
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
__device__ __forceinline__ void st32(uint32_t taddr, const float *r) {
  const uint32_t *u = reinterpret_cast<const uint32_t *>(r);
#pragma unroll
  for (int i = 0; i < 4; i++) st8(taddr + 8 * i, u + 8 * i);
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
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
__device__ __forceinline__ uint64_t add_2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// One step of this thread's row: 64 scores from tS, their weights over them. EDGE: some of the tile's rows don't see all
// of the step (pos: this row's last position, first: the step's first). m, l: the row's running maximum and sum.
template <int HP, bool HALF, bool EDGE>
__device__ __forceinline__ void softmax_step(uint32_t tS, uint32_t tO, const float4 *sc, float qf, int pos, int first,
                                             int j, float &m, float &l, uint64_t (*pv_done)[2], int *error) {
  float x[KT];
  ld32(tS, x);
  ld32(tS + 32, x + 32);
  float c[KU], lg[KU], inv[KU];
#pragma unroll
  for (int u = 0; u < KU; u++) {
    const float4 s = sc[u];
    c[u] = s.x * qf, lg[u] = s.y, inv[u] = s.z;
  }
  tmem_wait_ld();
  float most = -INFINITY;
#pragma unroll
  for (int u = 0; u < KU; u++) {
    if (EDGE) {
#pragma unroll
      for (int i = 0; i < UNIT; i++)
        if (first + u * UNIT + i > pos) x[u * UNIT + i] = -INFINITY;
    }
    float top = x[u * UNIT];
#pragma unroll
    for (int i = 1; i + 1 < UNIT; i += 2) top = max3(top, x[u * UNIT + i], x[u * UNIT + i + 1]);
    top = fmaxf(top, x[u * UNIT + UNIT - 1]);
    most = fmaxf(most, __fmaf_rn(top, c[u], lg[u]));
  }
  if (j == 0) {
    m = most;
  } else if (__any_sync(0xffffffffu, most > m + RESCALE)) {
    // O holds the steps so far: once the last P V is done, it and the sum go to the new maxima (the whole warp's rows:
    // TMEM is read and written by whole warps)
    mbar_wait(&(*pv_done)[(j - 1) & 1], ((j - 1) >> 1) & 1, error, 109);
    __syncwarp();
    fence_after();
    const float top = fmaxf(m, most), f = m == top ? 1.0f : ex2(m - top);
#pragma unroll
    for (int ch = 0; ch < HP / 32; ch++) {
      float o[32];
      ld32(tO + ch * 32, o);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; i++) o[i] *= f;
      st32(tO + ch * 32, o);
    }
    l *= f;
    m = top;
  }
  const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int u = 0; u < KU; u++) {
    const uint64_t c2 = f2(c[u], c[u]), a2 = f2(lg[u] - from, lg[u] - from);
    uint64_t sum = f2(0.0f, 0.0f);
    uint32_t hi[UNIT / 2], lo[UNIT / 2];
#pragma unroll
    for (int i = 0; i < UNIT; i += 2) {
      const uint64_t e = fma_2(f2(x[u * UNIT + i], x[u * UNIT + i + 1]), c2, a2);
      float w0 = ex2(lo_of(e)), w1 = ex2(hi_of(e));
      if (EDGE) {
        if (first + u * UNIT + i > pos) w0 = 0.0f;
        if (first + u * UNIT + i + 1 > pos) w1 = 0.0f;
      }
      sum = add_2(sum, f2(w0, w1));
      hi[i / 2] = pack(w0, w1);
      if (!HALF) {
        const float2 b = unpack(hi[i / 2]);
        lo[i / 2] = pack(w0 - b.x, w1 - b.y);
      }
    }
    // (a unit that the row does not see: 0 times a scale that may be NaN)
    l = __fmaf_rn(lo_of(sum) + hi_of(sum), !EDGE || first + u * UNIT <= pos ? inv[u] : 0.0f, l);
    st8(tS + 8 * u, hi);
    if (!HALF) st8(tS + 32 + 8 * u, lo);
  }
  wait_st();
}

template <int HP, bool HALF>
__global__ void __launch_bounds__(THREADS, 1) cache8_attention_tc_kernel(const Args a) {
  using S = Tc<HP, HALF>;
  constexpr int STAGES = S::STAGES, PARTS = S::PARTS;
  extern __shared__ uint8_t raw[];
  typename S::Smem &s = *reinterpret_cast<typename S::Smem *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  pdl_begin();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y;
  int *error = &a.meta[-1].y;

  // ---- which request's which pair of tiles
  int total = 0, fresh = 0;
  if (tid == 0) s.found[0] = -1;
  for (int base = 0; base < a.n_seqs; base += THREADS) {
    const int i = base + tid;
    int pairs = 0, own = 0;
    if (i < a.n_seqs) {
      const Request r = request_of(a, i);
      own = r.fresh;
      pairs = r.fresh * a.group > a.rows_most ? (r.fresh * a.group + 2 * QT - 1) / (2 * QT) : 0;
    }
    int upto = pairs;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    own = __reduce_add_sync(0xffffffffu, own);
    __syncthreads();
    if (lane == 31) s.part[0][warp] = upto, s.part[1][warp] = own;
    __syncthreads();
    int before = total;
    for (int w = 0; w < THREADS / 32; w++) {
      if (w < warp) before += s.part[0][w];
      total += s.part[0][w];
      fresh = min(fresh + s.part[1][w], a.n + 1);
    }
    const int x = (int)blockIdx.x - (before + upto - pairs);
    // the request's last pair, which sees the most positions, first
    if (x >= 0 && x < pairs) s.found[0] = i, s.found[1] = pairs - 1 - x;
  }
  if (fresh > a.n) return;  // starts that don't ascend
  __syncthreads();
  const int req = s.found[0], pair = s.found[1];
  if (req < 0) return;
  const Request r = request_of(a, req);
  const int rows = r.fresh * a.group, cap = a.width * a.block, row0 = pair * 2 * QT;
  // steps of each tile: up to its last row's position (and within the table's row)
  int steps[2];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int x = min(rows, row0 + (t + 1) * QT) - 1;  // the tile's last row
    const int seen = x < row0 + t * QT ? 0 : min(r.length - r.fresh + x / a.group + 1, cap);
    steps[t] = max(0, (seen + KT - 1) / KT);
  }
  const int most_steps = max(steps[0], steps[1]);

  if (tid == 0) {
    mbar_init(&s.q_full, 2 * QT);
    for (int i = 0; i < STAGES; i++) {
      mbar_init(&s.kv_full[i], QT);
      mbar_init(&s.kv_empty[i], 1);
    }
    for (int t = 0; t < 2; t++)
      for (int u = 0; u < 2; u++) {
        mbar_init(&s.s_full[t][u], 1);
        mbar_init(&s.p_full[t][u], 4);
        mbar_init(&s.pv_done[t][u], 1);
      }
    mbar_init(&s.mma_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem_base)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s.tmem_base;
  auto tS = [&](int t, int u) { return tmem + (uint32_t)(t * 2 * KT + u * KT); };
  auto tO = [&](int t) { return tmem + (uint32_t)(4 * KT + t * HP); };

  // (the launch's 512 x 128 registers: 128 x (96 + 176 + 176 + 56) = 512 x 126)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    // ---- the cache: thread tid brings 16 bytes of rows tid / CH + i * PER (CH pieces a row) of keys and of values
    constexpr int CH = HP / 16, PER = QT / CH, R = KT / PER;
    const int32_t *table = a.tables + (int64_t)req * a.width;
    const int piece = tid % CH, brow = tid / CH;
    const bool in_head = piece * 16 < a.hs;
    const int last_unit = min(cap, r.length) / UNIT;  // (units past it are no row's to see, or belong to NaN rows)
    auto page_of = [&](int u) { return u <= last_unit && u * UNIT < cap ? table[u * UNIT / a.block] : -1; };
    auto load = [&](const int8_t *cache, int j, int i, int page) {
      if (page < 0 || page >= a.blocks || !in_head) return make_uint4(0, 0, 0, 0);
      const int p = j * KT + brow + i * PER;
      return __ldg(reinterpret_cast<const uint4 *>(
          cache + (((int64_t)page * a.nkv + h) * a.block + p % a.block) * a.hs + piece * 16));
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
    int page[R], next[R];
    uint4 k[R], v[R];
    auto unit_of = [&](int j, int i) { return j * KU + (brow + i * PER) / UNIT; };
#pragma unroll
    for (int i = 0; i < R; i++) {
      page[i] = most_steps > 0 ? page_of(unit_of(0, i)) : -1;
      next[i] = most_steps > 1 ? page_of(unit_of(1, i)) : -1;
    }
#pragma unroll
    for (int i = 0; i < R; i++) k[i] = load(a.kc, 0, i, page[i]), v[i] = load(a.vc, 0, i, page[i]);
    // threads 0..3: a unit's scales, one step ahead, its block two
    int spage = -1;
    float ks = 0.0f, vs = 0.0f;
    auto scales = [&](int p) {
      const bool ok = p >= 0 && p < a.blocks;
      ks = ok ? a.ks[(int64_t)p * a.nkv + h] : __uint_as_float(0x7fffffffu);
      vs = ok ? a.vs[(int64_t)p * a.nkv + h] : __uint_as_float(0x7fffffffu);
    };
    if (tid < KU && most_steps > 0) {
      scales(page_of(tid));
      spage = most_steps > 1 ? page_of(KU + tid) : -1;
    }
    for (int j = 0; j < most_steps; j++) {
      const int slot = j % STAGES;
      if (!mbar_wait(&s.kv_empty[slot], ((j / STAGES) & 1) ^ 1, error, 101)) break;
      const bool more = j + 1 < most_steps;
#pragma unroll
      for (int i = 0; i < R; i++) {
        widened(s.k[slot][0], i, k[i]);
        if (more) k[i] = load(a.kc, j + 1, i, next[i]);
      }
#pragma unroll
      for (int i = 0; i < R; i++) {
        widened(s.v[slot][0], i, v[i]);
        if (more) v[i] = load(a.vc, j + 1, i, next[i]);
        next[i] = j + 2 < most_steps ? page_of(unit_of(j + 2, i)) : -1;
      }
      if (tid < KU) {
        // a key scale of 0 (a block of zeros) as the least: 0 times a masked -inf is no number
        const float c = !(ks * a.scale < 1e-30f) ? ks * a.scale : 1e-30f, w = !(vs < LEAST) ? vs : LEAST;
        s.sc[slot][tid] = make_float4(c, __log2f(w), __fdiv_rn(1.0f, w), 0.0f);
        if (more) {
          scales(spage);
          spage = j + 2 < most_steps ? page_of((j + 2) * KU + tid) : -1;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&s.kv_full[slot]);
    }
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 12) {
      const uint32_t id_s = idesc_f16(QT, KT), id_o = idesc_f16(QT, HP) | B_MAJOR_N;
      const int ksteps = a.hs / 16;
      auto issue_s = [&](int t, int j) {
        const int slot = j % STAGES;
        for (int part = 0; part < PARTS; part++)
          for (int kk = 0; kk < ksteps; kk++)
            mma_f16(tS(t, j & 1), desc_sw128(s.q[t][part][kk >> 2] + 32 * (kk & 3)),
                    desc_sw128(s.k[slot][kk >> 2] + 32 * (kk & 3)), id_s, part > 0 || kk > 0);
        mma_commit(&s.s_full[t][j & 1]);
      };
      auto issue_pv = [&](int t, int j) {
        const int slot = j % STAGES;
#pragma unroll
        for (int part = 0; part < PARTS; part++)
#pragma unroll
          for (int kk = 0; kk < KT / 16; kk++)
            mma_ts(tO(t), tS(t, j & 1) + 32 * part + 8 * kk, desc_head_major(s.v[slot][0] + 2048 * kk, KT * 128), id_o,
                   j > 0 || part > 0 || kk > 0);
        mma_commit(&s.pv_done[t][j & 1]);
      };
      bool ok = __all_sync(0xffffffffu, mbar_wait(&s.q_full, 0, error, 103));
      for (int j = 0; ok && j < 2 && j < most_steps; j++) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s.kv_full[j], 0, error, 104));
        if (!ok) break;
        fence_after();
        if (lane == 0)
          for (int t = 0; t < 2; t++)
            if (j < steps[t]) issue_s(t, j);
        __syncwarp();
      }
      for (int j = 0; ok && j < most_steps; j++) {
        const int ahead = (j + 2) % STAGES;
        for (int t = 0; ok && t < 2; t++) {
          if (j >= steps[t]) continue;
          ok = __all_sync(0xffffffffu, mbar_wait(&s.p_full[t][j & 1], (j >> 1) & 1, error, 106));
          if (!ok) break;
          fence_after();
          if (lane == 0) issue_pv(t, j);
          __syncwarp();
          if (j + 2 < steps[t]) {
            // (the scores' buffer holds P until P V is done)
            ok = mbar_wait(&s.pv_done[t][j & 1], (j >> 1) & 1, error, 107) &&
                 mbar_wait(&s.kv_full[ahead], ((j + 2) / STAGES) & 1, error, 108);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            if (lane == 0) issue_s(t, j + 2);
            __syncwarp();
          }
        }
        // every product that reads the stage is issued: it is free when they are done
        if (ok && lane == 0) mma_commit(&s.kv_empty[j % STAGES]);
        __syncwarp();
      }
      // every product issued has completed before the block frees TMEM
      if (lane == 0) mma_commit(&s.mma_done);
      __syncwarp();
      mbar_wait(&s.mma_done, 0, error, 114);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    // ---- the softmax of tile t: thread y has row row0 + t * QT + y, TMEM lane y
    const int t = (warp - 4) >> 2, y = tid - 128 * (t + 1), x = row0 + t * QT + y;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const bool on = x < rows;
    const int token = on ? x / a.group : 0, head = h * a.group + (on ? x % a.group : 0);
    const int pos = on ? r.length - r.fresh + token : -1;
    // its query, as float16 (float32: by a power of two into (0, 2), in two parts) in the swizzled layout
    float qf = 1.0f;
    {
      const int64_t off = (int64_t)(r.first + token) * a.q_stride + (int64_t)head * a.hs;
      float f = 1.0f;
      if (!HALF) {
        const float4 *src = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.q) + off);
        float top = 0.0f;
#pragma unroll 8
        for (int d = 0; d < a.hs / 4; d++) {
          const float4 z = on ? src[d] : make_float4(0, 0, 0, 0);
          top = fmaxf(fmaxf(fmaxf(top, fabsf(z.x)), fmaxf(fabsf(z.y), fabsf(z.z))), fabsf(z.w));
        }
        const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -126), 126);
        f = __uint_as_float((uint32_t)(127 - e) << 23);
        qf = __uint_as_float((uint32_t)(127 + e) << 23);
      }
#pragma unroll 4
      for (int d = 0; d < a.hs; d += 8) {
        uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
        if (on) {
          if (HALF) {
            hi = *reinterpret_cast<const uint4 *>(reinterpret_cast<const __half *>(a.q) + off + d);
          } else {
            const float4 *src = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.q) + off + d);
            const float4 z0 = src[0], z1 = src[1];
            const float z[8] = {z0.x * f, z0.y * f, z0.z * f, z0.w * f, z1.x * f, z1.y * f, z1.z * f, z1.w * f};
            uint32_t p[4], q[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
              p[i] = pack(z[2 * i], z[2 * i + 1]);
              const float2 b = unpack(p[i]);
              q[i] = pack(z[2 * i] - b.x, z[2 * i + 1] - b.y);
            }
            hi = make_uint4(p[0], p[1], p[2], p[3]), lo = make_uint4(q[0], q[1], q[2], q[3]);
          }
        }
        const int at = y * 128 + ((((d & 63) >> 3) ^ (y & 7)) << 4);
        *reinterpret_cast<uint4 *>(&s.q[t][0][d >> 6][at]) = hi;
        if (!HALF) *reinterpret_cast<uint4 *>(&s.q[t][PARTS - 1][d >> 6][at]) = lo;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&s.q_full);
    }
    const int first_pos = r.length - r.fresh + (row0 + t * QT) / a.group;  // the tile's first row's
    const uint32_t o_col = tO(t) + lane_base;
    float m = -INFINITY, l = 0.0f;
    const int n = steps[t];
    bool ok = true;
    for (int j = 0; j < n && ok; j++) {
      ok = mbar_wait(&s.s_full[t][j & 1], (j >> 1) & 1, error, 116);
      // (kv_full of this step completed before its scores: the scales, written before it, are there)
      ok = mbar_wait(&s.kv_full[j % STAGES], (j / STAGES) & 1, error, 117) && ok;
      ok = __all_sync(0xffffffffu, ok);
      fence_after();
      const float4 *sc = s.sc[j % STAGES];
      // (rows that don't exist have pos -1: nothing of a step is theirs, and nothing of theirs is written)
      if (j * KT + KT - 1 > first_pos)
        softmax_step<HP, HALF, true>(tS(t, j & 1) + lane_base, o_col, sc, qf, pos, j * KT, j, m, l, &s.pv_done[t], error);
      else
        softmax_step<HP, HALF, false>(tS(t, j & 1) + lane_base, o_col, sc, qf, pos, j * KT, j, m, l, &s.pv_done[t], error);
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.p_full[t][j & 1]);
    }
    if (n > 0) {
      ok = mbar_wait(&s.pv_done[t][(n - 1) & 1], ((n - 1) >> 1) & 1, error, 118) && ok;
      __syncwarp();
      fence_after();
    }
    float by = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    if (!ok || pos >= cap) by = __uint_as_float(0x7fffffffu);  // a wait gave up; a position past the table's row
    const int64_t off = (int64_t)(r.first + token) * a.out_stride + (int64_t)head * a.hs;
#pragma unroll
    for (int ch = 0; ch < HP / 32; ch++) {
      float o[32];
      __syncwarp();
      if (n > 0) {
        ld32(o_col + ch * 32, o);
        tmem_wait_ld();
      }
      if (!on) continue;
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        const int d = ch * 32 + i;
        if (d >= a.hs) break;
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] = n > 0 && by != 0.0f ? o[i + e] * by : by;
        if (HALF) {
          *reinterpret_cast<uint4 *>(reinterpret_cast<__half *>(a.out) + off + d) =
              make_uint4(pack(z[0], z[1]), pack(z[2], z[3]), pack(z[4], z[5]), pack(z[6], z[7]));
        } else {
          float4 *dst = reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.out) + off + d);
          dst[0] = make_float4(z[0], z[1], z[2], z[3]);
          dst[1] = make_float4(z[4], z[5], z[6], z[7]);
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 12) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int HP, bool HALF>
int launch_tc(const Args &a, cudaStream_t stream) {
  auto kernel = cache8_attention_tc_kernel<HP, HALF>;
  const size_t smem = sizeof(typename Tc<HP, HALF>::Smem) + 1024;
  B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  // pairs of tiles: all rows', and one more for every request that has any (at least rows_most + 1 rows each)
  const int64_t rows = (int64_t)a.n * a.group, requests = rows / (a.rows_most + 1);
  const int64_t pairs = rows / (2 * QT) + (requests < a.n_seqs ? requests : a.n_seqs);
  if (pairs < 1) return 0;
  launch(kernel, dim3((unsigned)pairs, a.nkv), dim3(THREADS), smem, stream, a);
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
