// cache8_attention.cu — attention over the paged 8-bit cache (cache8.cu), for single tokens and blocks of tokens of
// many requests at once: out = sum_j p_j v_j, p = softmax_j(q . k_j / sqrt(hs)) over the positions j up to the row's
// own, k_j = kscale[block][head] * int8, v_j likewise.
//
// A tile is RT (4, 8 or 16) query rows of one request and kv head: its tokens' query heads that share the kv head, so
// every byte of the cache is read once for all of them. Both products run on mma.sync with the cache as the 16-row
// operand; the scales stay outside (a block's key scale on its scores, its value scale within its weights), so the
// cache's values are never rounded.
//  - scores: the keys' bytes as they are (m16n8k32, signed bytes, exact int32 sums) with the queries in fixed point, each
//    row by a power of two into (0, 2) and then as four digits of a byte, 29 bits behind the point (a value is off by
//    2^-30 of its row's largest at most; with three digits an outlier of 1000 cost the others all below 2^-12 of their
//    size): a column for each digit of each row, whose sums are put together in float32.
//  - values: as float16 integers (exact), with the weights as a float16 pair high + low / 2^11, the low part taken so far up
//    that it keeps its 11 bits down to 2^-43 of the largest weight (float16 queries: one float16, half a step of the
//    output's type, down to 2^-31 of the largest).
//  - weights: w = 2^(s + log2(vscale) - M + 7), M a running maximum (per row) that moves only when it is passed by more
//    than 2^8, and the row sum l += w / vscale: the block's value scale costs no operation per value, and what is
//    rounded to float16 is relative to the largest term of the sum, whatever the scales.
// Work is split over the length of the caches: the tiles' units of 16 positions, laid end to end, are cut into equal
// spans, one for each thread block of a grid that fills the GPU once, so ragged requests balance and one long request
// takes every SM. A tile cut by a span's end leaves partial sums (unnormalized, with M and l) that combine_kernel
// joins in the order of the spans: results don't depend on timing.
// Loads: a warp copies a unit's rows by 16-byte pieces side by side (cp.async) into a ring of its own, so no warp waits for
// another. (Each lane copying what it will multiply itself, 64-byte runs of eight rows, read 4.5 TB/s, this 5.8.) The
// pieces of a row are swapped about by its number, so that neither the keys' reads nor the values' collide in a bank.
// Bound by reading the cache, and close behind by instructions. Measured, 32 query and 8 kv heads of 128: 64 requests of 512
// to 8192 positions, float32, 101 us (0.55 GB at 5.4 TB/s, 0.83 of a copy's rate; the loads by themselves 99); one of 131071,
// float16, 58 us (4.6 TB/s: 0.27 GB are read in 41 us, and the first loads, the cut at the end and the joining are 17 more).
#include <string>

#include "cache8.h"
#include "cache8_attention.cuh"

namespace b200 {
using namespace cache8;
namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int MOST_BLOCKS = 148 * 3;  // thread blocks of a grid (resident at once)
// A span's units at least, between what suits one request (fewer: more spans of it) and what suits several (more: less to
// join). Measured with 8, 16, 32 and 64 (32
// query and 8 kv heads of 128, float32): one request of 600 positions 10.4, 11.0, 12.6, 10.9 us, of 4000 13.9, 14.0, 15.5,
// 19.5, of 30,000 22.8, 22.9, 22.9, 26.8; 8 of 600 16.7, 17.2, 19.5, 12.5; 64 of 600 30.1, 30.3, 30.4, 26.8.
constexpr int MIN_UNITS = 32;

// Where a row's 16-byte piece q sits in the ring: 128-byte lines (of two rows of 64) with the pieces swapped by the row.
// The keys' reads take pieces 4 j + c of rows place(g), g = 2 i and 2 i + 1 at a time, the values' 16 (8) bytes g of rows
// place(2 c) or place(2 c + 1): each time in 128 bytes of different banks.
template <int HSEG>
__device__ __forceinline__ int piece_at(int row, int q) {
  if (HSEG == 1) return (row >> 1) * 128 + (((((row & 1) << 2) + q) ^ (row & 6)) << 4);
  return row * (HSEG == 2 ? 128 : 256) + (q >> 3) * 128 + (((q & 7) ^ (row & 7)) << 4);
}
// the position (of 8) that row g of a score tile stands for
template <int HSEG>
__device__ __forceinline__ int place(int g) {
  return HSEG == 1 ? g : g & 1 ? (g + 4) & 7 : g;
}

template <int RT>
__device__ __forceinline__ int tiles_of(const Args &a, const Request &r) {
  const int rows = r.fresh * a.group;
  return rows > a.rows_most ? 0 : (rows + RT - 1) / RT;
}
// its units: the positions that its table has room for, one unit at least (a row that sees nothing is written too)
__device__ __forceinline__ int units_of(const Args &a, const Request &r) {
  return max(1, (min(r.length, a.width * a.block) + UNIT - 1) / UNIT);
}

// BYTES (4 or 16) to shared memory
template <int BYTES>
__device__ __forceinline__ void copy(uint32_t dst, const void *src) {
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t interleave_lo(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5140); }
__device__ __forceinline__ uint32_t interleave_hi(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7362); }
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// D += A B of signed bytes, exact
__device__ __forceinline__ void mma_i8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four values of a query row
template <bool HALF>
__device__ __forceinline__ void query(const void *q, int64_t at, float (&z)[4]) {
  if (HALF) {
    const uint2 v = *reinterpret_cast<const uint2 *>(reinterpret_cast<const __half *>(q) + at);
    const float2 lo = unpack(v.x), hi = unpack(v.y);
    z[0] = lo.x, z[1] = lo.y, z[2] = hi.x, z[3] = hi.y;
  } else {
    const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(q) + at);
    z[0] = v.x, z[1] = v.y, z[2] = v.z, z[3] = v.w;
  }
}
// two float16 integers times 2^-11
__device__ __forceinline__ uint32_t lowered(uint32_t x) {
  const __half2 v = __hmul2(*reinterpret_cast<const __half2 *>(&x), __half2half2(__ushort_as_half(0x1000)));
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// sums of {work, tiles, requests astray} over the requests before this thread's (one request a thread), and of all
__device__ __forceinline__ void block_scan(int64_t (&v)[3], int64_t (&all)[3], int64_t (*part)[WARPS]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t own[3] = {v[0], v[1], v[2]};
#pragma unroll
  for (int j = 0; j < 3; j++)
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, v[j], d);
      if (lane >= d) v[j] += o;
    }
  __syncthreads();
  if (lane == 31) part[0][warp] = v[0], part[1][warp] = v[1], part[2][warp] = v[2];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 3; j++) {
    all[j] = 0;
    int64_t before = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      if (w < warp) before += part[j][w];
      all[j] += part[j][w];
    }
    v[j] += before - own[j];
  }
}

template <int HSEG, int RT, bool HALF>
struct Shape {
  static constexpr int HP = HSEG * 64;              // the head size, padded
  // Four rows of float32: the value products' eight columns hold the rows' weights' high parts and their low parts, so
  // one instruction does for both.
  static constexpr bool BOTH = RT == 4;
  static constexpr int NT = BOTH ? 1 : RT / 8;      // row tiles of the value products
  // the score products: 32 values of the head an instruction, columns by digit, then row
  static constexpr int KSTEPS = HSEG * 2, CT = RT / 2;
  static constexpr int VB = HSEG % 2 ? 8 : 16;      // bytes of a lane's piece of a value row
  static constexpr int VN = HP / (8 * VB);          // pieces
  static constexpr int ROW = HSEG <= 2 ? HP : 256;  // bytes of a row in the ring
  static constexpr int STAGE = 2 * UNIT * ROW;      // of a unit's keys and values
  static constexpr int RING = HSEG <= 2 ? 16384 : 24576;  // bytes of a warp's ring
  static constexpr int STAGES = RING / STAGE;       // 8, 4, 3, 3
  static constexpr int QREGS = KSTEPS * CT * 2;
  static constexpr bool QREG = QREGS <= 32;         // the query fragments in registers, else in shared memory
  static constexpr int MINB = HSEG * (BOTH ? 8 : RT) <= 16 ? 3 : 2;
  struct Smem {
    alignas(16) uint8_t ring[WARPS][RING];          // later the warps' sums [WARPS][RT][HP]
    alignas(16) uint2 qf[QREG ? 1 : KSTEPS * CT * 32];
    float sc[WARPS][STAGES][2];                     // the units' scales
    float ml[WARPS][RT][2];
    int64_t part[3][WARPS];
    int64_t found[3];
  };
};

// WHOLE: the head size is HSEG * 64 (copies then need no condition and only immediate offsets)
template <int HSEG, int RT, bool HALF, bool WHOLE>
__global__ void __launch_bounds__(THREADS, (Shape<HSEG, RT, HALF>::MINB)) cache8_attention_kernel(const Args a) {
  using S = Shape<HSEG, RT, HALF>;
  constexpr int NT = S::NT, HP = S::HP, STAGES = S::STAGES;
  constexpr bool BOTH = S::BOTH, PAIR = !HALF && !BOTH;  // PAIR: the low parts in instructions of their own
  const int hs = WHOLE ? HP : a.hs;
  extern __shared__ __align__(16) uint8_t raw[];
  typename S::Smem &sm = *reinterpret_cast<typename S::Smem *>(raw);
  pdl_begin();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int h = blockIdx.y;

  // ---- this block's span of the work, and the request in which it begins; {work, tiles} before that request. Work is
  // units, or, where no tile is longer than a span has to be, tiles (none is cut then).
  int64_t before[2] = {0, 0};
  int64_t v[3], all[3], sum[3] = {0, 0, 0}, w = 0;
  auto add_up = [&](int base) {
    const int i = base + tid;
    v[0] = v[1] = v[2] = w = 0;
    if (i < a.n_seqs) {
      const Request r = request_of(a, i);
      v[2] = r.astray;
      v[1] = tiles_of<RT>(a, r);
      w = v[0] = v[1] * (a.whole_tiles ? 1 : units_of(a, r));
    }
    block_scan(v, all, sm.part);
  };
  for (int base = 0; base < a.n_seqs; base += THREADS) {
    add_up(base);
#pragma unroll
    for (int j = 0; j < 3; j++) sum[j] += all[j];
  }
  // (starts that don't ascend: nothing is written)
  const int64_t total = sum[2] ? 0 : sum[0];
  const int64_t span = max((int64_t)a.min_work, (total + gridDim.x - 1) / gridDim.x);
  int64_t at = span * blockIdx.x;
  const int64_t end = min(at + span, total);
  if (blockIdx.x == 0 && h == 0 && tid == 0) a.meta[-1] = make_int4(total ? (int)sum[1] : 0, 0, 0, 0);
  if (at >= end) return;
  int64_t carry[2] = {0, 0};
  for (int base = 0; base < a.n_seqs; base += THREADS) {
    if (a.n_seqs > THREADS) add_up(base);
    if (w && carry[0] + v[0] <= at && at < carry[0] + v[0] + w) {
      sm.found[0] = carry[0] + v[0];
      sm.found[1] = carry[1] + v[1];
      sm.found[2] = base + tid;
    }
    carry[0] += all[0], carry[1] += all[1];
  }
  __syncthreads();
  before[0] = sm.found[0], before[1] = sm.found[1];
  int req = (int)sm.found[2];

  const int page_bytes = a.nkv * a.block * hs;
  const int step_blocks = WARPS * UNIT / a.block, step_rest = WARPS * UNIT % a.block;  // a warp's way to its next unit
  const uint32_t ring = smem_addr(sm.ring[warp]);
  uint8_t *ring_p = sm.ring[warp];
  while (at < end) {
    const Request r = request_of(a, req);
    const int tiles = tiles_of<RT>(a, r), units = units_of(a, r);
    if (tiles == 0) {
      req++;
      continue;
    }
    const int per_tile = a.whole_tiles ? 1 : units;
    const int tile = (int)((at - before[0]) / per_tile), begin = (int)((at - before[0]) % per_tile);
    const int stop = (int)min((int64_t)per_tile, begin + (end - at));
    const int u0 = begin, u1 = a.whole_tiles ? units : stop;
    const int64_t tile_at = before[0] + (int64_t)tile * per_tile;
    const int span0 = (int)(tile_at / span), spans = (int)((tile_at + per_tile - 1) / span) - span0 + 1;
    const int64_t tile_id = before[1] + tile;
    if (h == 0 && tid == 0 && begin == 0) a.meta[tile_id] = make_int4(span0, spans, req, tile);

    // ---- the tile's rows: row x is query head x % group of the kv head, of the request's token x / group
    const int rows = r.fresh * a.group, x0 = tile * RT, cap = a.width * a.block;
    const int last = r.length - r.fresh + (min(rows, x0 + RT) - 1) / a.group;  // the last row's position
    const int first = r.length - r.fresh + x0 / a.group;                       // the first row's
    const int u_end = min(u1, (min(last + 1, cap) + UNIT - 1) / UNIT);         // no row sees further units

    // this lane's places in the ring: of the pieces it copies, and of those it multiplies (of the first half of the rows)
    int piece_to[HSEG * 2];
#pragma unroll
    for (int i = 0; i < HSEG * 2; i++) {
      const int piece = i * 32 + lane, per = WHOLE ? HSEG * 4 : hs / 16;
      piece_to[i] = piece_at<HSEG>(piece / per, piece % per);
    }
    const int k_from = piece_at<HSEG>(place<HSEG>(g), c);
    const int v_from[2] = {piece_at<HSEG>(place<HSEG>(2 * c), S::VB == 16 ? g : g >> 1) + (S::VB == 16 ? 0 : (g & 1) * 8),
                           piece_at<HSEG>(place<HSEG>(2 * c + 1), S::VB == 16 ? g : g >> 1) + (S::VB == 16 ? 0 : (g & 1) * 8)};
    // The ring's front: the next unit to copy, its block's place in the table and its place in the block, and the id of
    // that block (read one unit ahead).
    const int32_t *table = a.tables + (int64_t)req * a.width;
    int front = u0 + warp, front_block = front * UNIT / a.block, front_at = front * UNIT % a.block;
    auto forward = [&]() {
      front += WARPS;
      front_block += step_blocks, front_at += step_rest;
      if (front_at >= a.block) front_at -= a.block, front_block++;
    };
    auto front_page = [&]() { return front < u_end ? table[front_block] : -1; };
    // (the first units' at once: a lane a unit)
    const int ids = front + lane * WARPS < u_end && lane < STAGES ? table[(front + lane * WARPS) * UNIT / a.block] : -1;
    int page = __shfl_sync(0xffffffffu, ids, 0);
    const int8_t *k_lane = a.kc + (int64_t)h * a.block * hs + lane * 16;
    const int8_t *v_lane = a.vc + (int64_t)h * a.block * hs + lane * 16;
    const float *s_lane = (lane == 1 ? a.vs : a.ks) + h;
    auto issue = [&](int slot, auto &&next_page) {
      const int mine = page, at = front_at;
      const bool there = front < u_end, ok = (uint32_t)mine < (uint32_t)a.blocks;
      forward();
      page = next_page();
      if (there) {
        if (ok) {
          const int64_t off = (int64_t)mine * page_bytes + at * hs;
          const int8_t *k = k_lane + off, *v = v_lane + off;
          const uint32_t dst = ring + slot * S::STAGE;
#pragma unroll
          for (int i = 0; i < HSEG * 2; i++)
            if (WHOLE || i * 32 + lane < hs) copy<16>(dst + piece_to[i], k + i * 512);
#pragma unroll
          for (int i = 0; i < HSEG * 2; i++)
            if (WHOLE || i * 32 + lane < hs) copy<16>(dst + UNIT * S::ROW + piece_to[i], v + i * 512);
        }
        // a table entry that is no block of the pool: NaN scales, so every row that sees it comes out NaN
        if (lane < 2) {
          float *dst_s = &sm.sc[warp][slot][lane];
          if (ok) copy<4>(smem_addr(dst_s), s_lane + (int64_t)mine * a.nkv);
          else *dst_s = __uint_as_float(0x7fffffffu);
        }
      }
      copies_commit();
    };
    __syncthreads();  // (the tile before has left the ring)
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) issue(s, [&]() { return __shfl_sync(0xffffffffu, ids, s + 1); });

    // this lane's column p of row tile t, as a row of the tile
    auto row_of = [&](int t, int p) { return BOTH ? 2 * (c & 1) + p : 8 * t + 2 * c + p; };
    // Query fragments: lane (g, c) holds column 8 t + g of column tile t, digit (8 t + g) / RT of row (8 t + g) % RT, of the
    // head's values 64 j + 16 c .. + 15, the bytes of keys that it copies.
    uint32_t qd[S::QREG ? S::KSTEPS * S::CT : 1][2];
    float qf[NT][2];  // what the scores of this lane's columns (rows 2 c, 2 c + 1 of row tile t) are to be scaled by
    {
      float f[NT], back[NT];
      int64_t off[NT];
      bool is[NT];
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const int x = x0 + (BOTH ? g & 3 : 8 * t + g);
        is[t] = x < rows;
        off[t] = (int64_t)(r.first + (is[t] ? x / a.group : 0)) * a.q_stride + (int64_t)(h * a.group + (is[t] ? x % a.group : 0)) * hs;
        // each row by a power of two into (0, 2)
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < HSEG; j++)
          if (is[t] && (WHOLE || 64 * j + 16 * c < hs)) {
#pragma unroll
            for (int w = 0; w < 4; w++) {
              float z[4];
              query<HALF>(a.q, off[t] + 64 * j + 16 * c + 4 * w, z);
#pragma unroll
              for (int i = 0; i < 4; i++) top = max(top, __float_as_uint(z[i]) & 0x7fffffffu);
            }
          }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // (rows below 2^-90 as if they were of that size: what they are scaled back by stays a whole float32; 2^-127, for
        // the largest, is a subnormal)
        const int e = min(max((int)(top >> 23) - 127, -90), 127);
        f[t] = __uint_as_float(max((uint32_t)(127 - e) << 23, 0x400000u));
        back[t] = __uint_as_float((uint32_t)(127 + e) << 23) * 1.862645149230957e-9f;  // 2^-29
        if (top >= 0x7f800000u) back[t] = __uint_as_float(0x7fffffffu);  // (a row with an infinity or a NaN: NaN)
        qf[t][0] = __shfl_sync(0xffffffffu, back[t], BOTH ? 8 * (c & 1) : 8 * c) * a.scale;
        qf[t][1] = __shfl_sync(0xffffffffu, back[t], BOTH ? 8 * (c & 1) + 4 : 8 * c + 4) * a.scale;
      }
      auto keep = [&](int k, uint32_t first, uint32_t then) {
        if (S::QREG) qd[S::QREG ? k : 0][0] = first, qd[S::QREG ? k : 0][1] = then;
        else if (warp == 0) sm.qf[S::QREG ? 0 : k * 32 + lane] = make_uint2(first, then);
      };
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < S::KSTEPS; i++) {
          uint32_t word[4][2] = {};
          const int d = 64 * (i / 2) + 16 * c + 8 * (i & 1);
          if (is[t] && (WHOLE || d < hs)) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
              float z[4];
              query<HALF>(a.q, off[t] + d + 4 * y, z);
#pragma unroll
              for (int e = 0; e < 4; e++) {
                // q 2^29 = 2^24 d0 + 2^16 d1 + 2^8 d2 + d3, the digits from -128 to 127: with 128 added to the lower
                // three, the bytes of the sum, less that
                const uint32_t sum = ((uint32_t)__float2int_rn(z[e] * f[t] * 536870912.0f) + 0x808080u) ^ 0x808080u;
#pragma unroll
                for (int k = 0; k < 4; k++) word[k][y] |= (sum >> (24 - 8 * k) & 255) << (8 * e);
              }
            }
          }
          if (BOTH) {
            keep(i * S::CT, g < 4 ? word[0][0] : word[1][0], g < 4 ? word[0][1] : word[1][1]);
            keep(i * S::CT + 1, g < 4 ? word[2][0] : word[3][0], g < 4 ? word[2][1] : word[3][1]);
          } else {
#pragma unroll
            for (int k = 0; k < 4; k++) keep((i * S::CT + k * NT + t) % (S::KSTEPS * S::CT), word[k][0], word[k][1]);
          }
        }
    }
    int pos[NT][2];  // the positions of this lane's columns (-1: no row)
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int p = 0; p < 2; p++) {
        const int x = x0 + row_of(t, p);
        pos[t][p] = x < rows ? r.length - r.fresh + x / a.group : -1;
      }
    if (!S::QREG) __syncthreads();

    // ---- the units of this warp: u0 + warp, + WARPS, ...
    float M[NT][2], from[NT][2], l[NT][2], o[NT][HSEG * 4][4];  // (from: M less LIFT, or 0 while that is -inf)
#pragma unroll
    for (int t = 0; t < NT; t++) {
      M[t][0] = M[t][1] = -INFINITY;
      l[t][0] = l[t][1] = from[t][0] = from[t][1] = 0.0f;
#pragma unroll
      for (int m = 0; m < HSEG * 4; m++) o[t][m][0] = o[t][m][1] = o[t][m][2] = o[t][m][3] = 0.0f;
    }
    // raw scores of the unit in a slot: S^T = K Q^T, 16 positions x 8 columns an instruction
    auto score = [&](int slot, int (&si)[S::CT][4]) {
#pragma unroll
      for (int t = 0; t < S::CT; t++) si[t][0] = si[t][1] = si[t][2] = si[t][3] = 0;
      const uint8_t *base = ring_p + slot * S::STAGE;
#pragma unroll
      for (int j = 0; j < HSEG; j++) {
        const uint8_t *row = base + (j >> 1) * 128 + (k_from ^ ((j & 1) << 6));
        const uint4 k0 = *reinterpret_cast<const uint4 *>(row);
        const uint4 k1 = *reinterpret_cast<const uint4 *>(row + 8 * S::ROW);
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
          for (int t = 0; t < S::CT; t++) {
            const int k = (2 * j + w) * S::CT + t;
            uint2 q;
            if (S::QREG) q = make_uint2(qd[S::QREG ? k : 0][0], qd[S::QREG ? k : 0][1]);
            else q = sm.qf[S::QREG ? 0 : k * 32 + lane];
            if (w == 0) mma_i8(si[t], k0.x, k1.x, k0.y, k1.y, q.x, q.y);
            else mma_i8(si[t], k0.z, k1.z, k0.w, k1.w, q.x, q.y);
          }
      }
    };
    // The next unit's scores are worked out beside this unit's weights and values: neither waits for the other, and with
    // three warps a scheduler it is waiting for one instruction after the other that takes the time.
    if (u0 + warp < u_end) {
      copies_wait<STAGES - 2>();
      __syncwarp();
      int si[S::CT][4];
      score(0, si);
      int slot = 0;
#pragma unroll 1
      for (int u = u0 + warp; u < u_end; u += WARPS) {
        const int after = slot + 1 == STAGES ? 0 : slot + 1;
        copies_wait<STAGES - 3>();
        __syncwarp();  // (every lane is through with the slot before this one, which is refilled at once)
        issue(slot == 0 ? STAGES - 1 : slot - 1, front_page);
        const float kscale = sm.sc[warp][slot][0], vscale = sm.sc[warp][slot][1];
        const uint8_t *base = ring_p + slot * S::STAGE;
        int next[S::CT][4];
        score(after, next);  // (of the last unit: of what the slot held, for nothing)
        float s[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if (BOTH) {
              // lanes c < 2 have the first and the third digits, c >= 2 the second and the last ones, of the same rows
              const float v = (float)si[0][e] * (c < 2 ? 16777216.0f : 65536.0f) + (float)si[1][e] * (c < 2 ? 256.0f : 1.0f);
              s[t][e] = v + __shfl_xor_sync(0xffffffffu, v, 2);
            } else {
              s[t][e] = __fmaf_rn((float)si[(2 * NT + t) % S::CT][e], 256.0f, (float)si[(3 * NT + t) % S::CT][e]);
              s[t][e] = __fmaf_rn((float)si[(NT + t) % S::CT][e], 65536.0f, s[t][e]);
              s[t][e] = __fmaf_rn((float)si[t][e], 16777216.0f, s[t][e]);
            }
          }
        // ---- weights. A value scale below 2^-92 counts as 2^-92 (a block of zeros has scale 0): what it weighs
        // is below any other block's last place
        const float vs = !(vscale < LEAST) ? vscale : LEAST;
        const float lg = __log2f(vs), inv = __frcp_rn(vs);
        float f[NT][2], y[NT][4];  // (the exponents, as far as the maximum is concerned)
        bool up = false;
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
          for (int p = 0; p < 2; p++) f[t][p] = kscale * qf[t][p];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            y[t][e] = __fmaf_rn(s[t][e], f[t][e & 1], lg);
          }
        }
        const bool masked = u * UNIT + UNIT - 1 > first;
        auto sees = [&](int t, int e) { return u * UNIT + place<HSEG>(g) + 8 * (e >> 1) <= pos[t][e & 1]; };
        if (masked) {
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) y[t][e] = sees(t, e) ? y[t][e] : -INFINITY;
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int p = 0; p < 2; p++) up |= fmaxf(y[t][p], y[t][2 + p]) > M[t][p] + RESCALE;
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
              float m = fmaxf(y[t][p], y[t][2 + p]);
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              m = fmaxf(m, M[t][p]);
              const float by = M[t][p] == m ? 1.0f : ex2(M[t][p] - m);
              l[t][p] *= by;
#pragma unroll
              for (int x = 0; x < HSEG * 4; x++) o[t][x][p] *= by, o[t][x][2 + p] *= by;
              M[t][p] = m;
              from[t][p] = m == -INFINITY ? 0.0f : m - LIFT;
            }
        }
        uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
          float w[4], by[2] = {inv, inv};
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = ex2(__fmaf_rn(s[t][e], f[t][e & 1], lg - from[t][e & 1]));
          if (masked) {
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = sees(t, e) ? w[e] : 0.0f;
            // (a row that sees nothing of the unit: 0 times a scale that may be NaN)
#pragma unroll
            for (int p = 0; p < 2; p++) by[p] = sees(t, p) ? inv : 0.0f;
          }
          l[t][0] = __fmaf_rn(w[0] + w[2], by[0], l[t][0]);
          l[t][1] = __fmaf_rn(w[1] + w[3], by[1], l[t][1]);
#pragma unroll
          for (int x = 0; x < 2; x++) {
            uint32_t hi = pack(w[2 * x], w[2 * x + 1]), lo = 0;
            if (!HALF) {
              const float2 b = unpack(hi);
              lo = pack((w[2 * x] - b.x) * 2048.0f, (w[2 * x + 1] - b.y) * 2048.0f);
            }
            ph[t][x] = transposed(BOTH && c >= 2 ? lo : hi);
            if (PAIR) pl[t][x] = transposed(lo);
          }
        }
        // ---- O^T += V^T P^T: lane (g, c)'s pieces of the rows place(2 c), place(2 c + 1), and 8 on
        const uint8_t *vbase = base + UNIT * S::ROW;
#pragma unroll
        for (int p = 0; p < S::VN; p++) {
          uint32_t vw[4][S::VB / 4];
#pragma unroll
          for (int y = 0; y < 4; y++) {
            // piece (8 p + g) of 16 bytes, or 8 bytes 8 p + g
            const uint8_t *src = vbase + (y >> 1) * 8 * S::ROW +
                                 (S::VB == 16 ? p * 128 + v_from[y & 1] : (p >> 1) * 128 + (v_from[y & 1] ^ ((p & 1) << 6)));
            if (S::VB == 16) {
              const uint4 v = *reinterpret_cast<const uint4 *>(src);
              vw[y][0] = v.x, vw[y][1] = v.y, vw[y][S::VB / 4 - 2] = v.z, vw[y][S::VB / 4 - 1] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2 *>(src);
              vw[y][0] = v.x, vw[y][1] = v.y;
            }
          }
#pragma unroll
          for (int w = 0; w < S::VB / 4; w++) {
            uint32_t a0[2], a1[2], a2[2], a3[2];
#pragma unroll
            for (int y = 0; y < 2; y++) {
              const uint32_t p0 = (y ? interleave_hi(vw[0][w], vw[1][w]) : interleave_lo(vw[0][w], vw[1][w])) ^ 0x80808080u;
              const uint32_t p1 = (y ? interleave_hi(vw[2][w], vw[3][w]) : interleave_lo(vw[2][w], vw[3][w])) ^ 0x80808080u;
              a0[y] = widen<0x4140>(p0), a1[y] = widen<0x4342>(p0), a2[y] = widen<0x4140>(p1), a3[y] = widen<0x4342>(p1);
            }
            const int m = p * S::VB / 2 + 2 * w;
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
              for (int y = 0; y < 2; y++) mma(o[t][m + y], a0[y], a1[y], a2[y], a3[y], ph[t][0], ph[t][1]);
            }
            if (PAIR) {
              // (the values go down by as much as the low parts went up, which is exact)
#pragma unroll
              for (int y = 0; y < 2; y++) {
                a0[y] = lowered(a0[y]), a1[y] = lowered(a1[y]), a2[y] = lowered(a2[y]), a3[y] = lowered(a3[y]);
#pragma unroll
                for (int t = 0; t < NT; t++) mma(o[t][m + y], a0[y], a1[y], a2[y], a3[y], pl[t][0], pl[t][1]);
              }
            }
          }
        }
#pragma unroll
        for (int t = 0; t < S::CT; t++)
#pragma unroll
          for (int e = 0; e < 4; e++) si[t][e] = next[t][e];
        slot = after;
      }
    }
    copies_wait<0>();

    // ---- the four warps' sums to one M a row, then added in the warps' order
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int p = 0; p < 2; p++) {
        l[t][p] += __shfl_xor_sync(0xffffffffu, l[t][p], 4);
        l[t][p] += __shfl_xor_sync(0xffffffffu, l[t][p], 8);
        l[t][p] += __shfl_xor_sync(0xffffffffu, l[t][p], 16);
        if (g == 0) sm.ml[warp][row_of(t, p)][0] = M[t][p], sm.ml[warp][row_of(t, p)][1] = l[t][p];
      }
    if (BOTH) {
#pragma unroll
      for (int m = 0; m < HSEG * 4; m++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[0][m][e] += 4.8828125e-4f * __shfl_xor_sync(0xffffffffu, o[0][m][e], 2);  // 2^-11
    }
    __syncthreads();
    float *sums = reinterpret_cast<float *>(sm.ring);
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int p = 0; p < 2; p++) {
        const int x = row_of(t, p);
        float top = sm.ml[0][x][0];
#pragma unroll
        for (int w = 1; w < WARPS; w++) top = fmaxf(top, sm.ml[w][x][0]);
        const float by = M[t][p] == top ? 1.0f : ex2(M[t][p] - top);
        float *dst = sums + ((int64_t)warp * RT + x) * HP;
#pragma unroll
        for (int q = 0; q < S::VN; q++)
#pragma unroll
          for (int w = 0; w < S::VB / 4; w++) {
            const int m = q * S::VB / 2 + 2 * w;
            if (!BOTH || c < 2) *reinterpret_cast<float4 *>(dst + q * 8 * S::VB + S::VB * g + 4 * w) = make_float4(
                o[t][m][p] * by, o[t][m][2 + p] * by, o[t][m + 1][p] * by, o[t][m + 1][2 + p] * by);
          }
      }
    __syncthreads();
    const int quads = hs / 4;
    for (int i = tid; i < RT * quads; i += THREADS) {
      const int x = i / quads, d = (i - x * quads) * 4;
      if (x0 + x >= rows) break;
      float top = sm.ml[0][x][0], sum_l = 0.0f;
#pragma unroll
      for (int w = 1; w < WARPS; w++) top = fmaxf(top, sm.ml[w][x][0]);
      float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        const float m = sm.ml[w][x][0];
        sum_l += sm.ml[w][x][1] * (m == top ? 1.0f : ex2(m - top));
        const float4 v = *reinterpret_cast<const float4 *>(sums + ((int64_t)w * RT + x) * HP + d);
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
      const int token = (x0 + x) / a.group, head = h * a.group + (x0 + x) % a.group;
      if (r.length - r.fresh + token >= cap) sum_l = __uint_as_float(0x7fffffffu);  // positions past the table's row
      if (spans == 1) {
        const float by = sum_l == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum_l);
        const int64_t off = (int64_t)(r.first + token) * a.out_stride + (int64_t)head * hs + d;
        if (HALF) {
          *reinterpret_cast<uint2 *>(reinterpret_cast<__half *>(a.out) + off) =
              make_uint2(pack(sum.x * by, sum.y * by), pack(sum.z * by, sum.w * by));
        } else {
          *reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.out) + off) =
              make_float4(sum.x * by, sum.y * by, sum.z * by, sum.w * by);
        }
      } else {
        const int64_t row = ((blockIdx.x + tile_id) * a.nkv + h) * RT + x;
        *reinterpret_cast<float4 *>(a.part + row * hs + d) = sum;
        if (d == 0) a.part_ml[row] = make_float2(top, sum_l);
      }
    }
    at += stop - begin;
    if (tile + 1 == tiles && stop == per_tile) {
      before[0] += (int64_t)tiles * per_tile;
      before[1] += tiles;
      req++;
    }
  }
}

// The rows of tiles that several spans have worked on: the partial sums joined, a row by SHARE warps, each in the spans'
// order, and those in theirs. SHARE 4 where there are few tiles (then it is the many spans of a long request that take
// time), else 1.
constexpr int CW = 4;  // warps
template <int RT, int SHARE, bool HALF>
__global__ void __launch_bounds__(CW * 32) cache8_combine_kernel(const Args a) {
  pdl_begin();
  constexpr int ROWS = CW / SHARE;  // rows at a time
  __shared__ float acc[CW][256], ml[CW][2];
  const int tile_id = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp % SHARE;
  if (tile_id >= a.meta[-1].x) return;
  const int4 meta = a.meta[tile_id];
  if (meta.y < 2) return;
  const Request r = request_of(a, meta.z);
  for (int x0 = blockIdx.z * ROWS; x0 < RT; x0 += gridDim.z * ROWS) {
    const int x = x0 + warp / SHARE, row_of = meta.w * RT + x;
    if (meta.w * RT + x0 >= r.fresh * a.group) break;
    const bool on = row_of < r.fresh * a.group;
    float M = -INFINITY, l = 0.0f;
    float4 o[2];  // this lane's values 4 lane .. + 3, and 128 on
    o[0] = o[1] = make_float4(0, 0, 0, 0);
#pragma unroll 2
    for (int s = part; s < meta.y && on; s += SHARE) {
      const int64_t row = (((int64_t)meta.x + s + tile_id) * a.nkv + h) * RT + x;
      const float2 v = a.part_ml[row];
      float4 z[2];
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (4 * lane + 128 * j < a.hs) z[j] = *reinterpret_cast<const float4 *>(a.part + row * a.hs + 4 * lane + 128 * j);
      const float m = fmaxf(M, v.x), by = M == m ? 1.0f : ex2(M - m), vy = v.x == m ? 1.0f : ex2(v.x - m);
      l = l * by + v.y * vy;
      M = m;
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (4 * lane + 128 * j < a.hs) {
          o[j].x = o[j].x * by + z[j].x * vy, o[j].y = o[j].y * by + z[j].y * vy;
          o[j].z = o[j].z * by + z[j].z * vy, o[j].w = o[j].w * by + z[j].w * vy;
        }
    }
    if (SHARE > 1) {
      if (lane == 0) ml[warp][0] = M, ml[warp][1] = l;
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (4 * lane + 128 * j < a.hs) *reinterpret_cast<float4 *>(&acc[warp][4 * lane + 128 * j]) = o[j];
      __syncthreads();
      float top = ml[warp - part][0];
#pragma unroll
      for (int w = 1; w < SHARE; w++) top = fmaxf(top, ml[warp - part + w][0]);
      l = 0.0f;
      o[0] = o[1] = make_float4(0, 0, 0, 0);
      if (part == 0) {
#pragma unroll
        for (int w = 0; w < SHARE; w++) {
          const float m = ml[warp + w][0], by = m == top ? 1.0f : ex2(m - top);
          l += ml[warp + w][1] * by;
#pragma unroll
          for (int j = 0; j < 2; j++)
            if (4 * lane + 128 * j < a.hs) {
              const float4 z = *reinterpret_cast<const float4 *>(&acc[warp + w][4 * lane + 128 * j]);
              o[j].x += z.x * by, o[j].y += z.y * by, o[j].z += z.z * by, o[j].w += z.w * by;
            }
        }
      }
    }
    if (part == 0 && on) {
      const float f = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
      const int token = row_of / a.group, head = h * a.group + row_of % a.group;
      const int64_t off = (int64_t)(r.first + token) * a.out_stride + (int64_t)head * a.hs + 4 * lane;
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (4 * lane + 128 * j < a.hs) {
          if (HALF)
            *reinterpret_cast<uint2 *>(reinterpret_cast<__half *>(a.out) + off + 128 * j) =
                make_uint2(pack(o[j].x * f, o[j].y * f), pack(o[j].z * f, o[j].w * f));
          else
            *reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.out) + off + 128 * j) =
                make_float4(o[j].x * f, o[j].y * f, o[j].z * f, o[j].w * f);
        }
    }
    if (SHARE > 1) __syncthreads();  // acc and ml have been read
  }
}
template <int RT, bool HALF>
int launch_combine(const Args &a, int64_t tiles, cudaStream_t stream) {
  // (measured, by four warps and by one: one request of 130,000 positions 56 and 66 us, of 8000 17 and 19.6; 64 of 4000 94
  // and 92)
  const bool few = tiles * a.nkv <= 64;
  const dim3 grid((unsigned)tiles, a.nkv, few ? RT : 1);
  launch(few ? cache8_combine_kernel<RT, CW, HALF> : cache8_combine_kernel<RT, 1, HALF>, grid, dim3(CW * 32), 0, stream, a);
  B200_LAUNCHED("cache8_combine");
  return 0;
}

// rows of a tile: 8 where the requests have that few on average (float32: 4, see Shape), else 16 (a row tile costs
// instructions whether its rows are there or not; a request with more rows takes several tiles). The average is of the
// buffers' rows, n. Measured with 64 single tokens over 600 to 8000 positions, 4 query heads a kv head, float32: n = 64
// (4 rows a tile) 107 us, 65 to 128 (8) 132, 256 (16) 206, 4096 232; float16 n = 64 to 128 (8) 118 to 126, 256 (16) 179.
int rows_of_tile(int n, int n_seqs, int group, bool half) {
  const int64_t rows = (int64_t)n * group;
  return !half && rows <= 4 * (int64_t)n_seqs ? 4 : rows <= 8 * (int64_t)n_seqs ? 8 : 16;
}

// The scratch: as much as any tile height of up to 16 takes, so that it never shrinks as n or n_seqs grow (rows_of_tile goes
// up with one and down with the other), and a scratch for the most of both serves every call of no more.
struct Layout {
  int rt;
  int64_t tiles;
  uint64_t ml_at, part_at, bytes;
};
Layout layout_of(int n, int n_seqs, int nh, int nkv, int hs, bool half) {
  Layout s;
  const int group = nh / nkv;
  s.rt = rows_of_tile(n, n_seqs, group, half);
  const int64_t rows = (int64_t)n * group, requests = n < n_seqs ? n : n_seqs;
  s.tiles = (rows + s.rt - 1) / s.rt + requests;
  // rows of partial sums: those of (tiles + spans) tiles, of 4 rows as of 16
  const uint64_t parts = (rows + 16 * (1 + requests + (MOST_BLOCKS + nkv - 1) / nkv)) * nkv;
  const auto up = [](uint64_t x) { return (x + 255) / 256 * 256; };
  s.ml_at = up(((rows + 3) / 4 + requests + 1) * sizeof(int4));
  s.part_at = s.ml_at + up(parts * sizeof(float2));
  s.bytes = s.part_at + up(parts * (uint64_t)hs * sizeof(float));
  return s;
}

template <int HSEG, int RT, bool HALF, bool WHOLE>
int launch_attention8(const Args &a, int blocks_x, cudaStream_t stream) {
  using S = Shape<HSEG, RT, HALF>;
  auto kernel = cache8_attention_kernel<HSEG, RT, HALF, WHOLE>;
  B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(typename S::Smem)));
  const int most = a.whole_tiles ? blocks_x : 148 * S::MINB / a.nkv;
  launch(kernel, dim3(most < 1 ? 1 : most < blocks_x ? most : blocks_x, a.nkv), dim3(THREADS), sizeof(typename S::Smem),
         stream, a);
  B200_LAUNCHED("cache8_attention");
  return 0;
}
using Launch = int (*)(const Args &, int, cudaStream_t);
template <int HSEG, int RT>
Launch launch_of(bool half, bool whole) {
  if (half) return whole ? launch_attention8<HSEG, RT, true, true> : launch_attention8<HSEG, RT, true, false>;
  return whole ? launch_attention8<HSEG, RT, false, true> : launch_attention8<HSEG, RT, false, false>;
}
template <int HSEG>
Launch launch_of(int rt, bool half, bool whole) {
  if (rt == 4) return whole ? launch_attention8<HSEG, 4, false, true> : launch_attention8<HSEG, 4, false, false>;
  return rt == 8 ? launch_of<HSEG, 8>(half, whole) : launch_of<HSEG, 16>(half, whole);
}

int check_sizes(const char *what, int n, int n_seqs, int nh, int nkv, int hs) {
  const std::string name(what);
  if (n < 0 || n_seqs < 1 || n_seqs > 65536) return fail(B200FWD_EINVAL, name + ": 1 to 65536 requests, no fewer than 0 tokens");
  if (nkv < 1 || nh < nkv || nh % nkv || nkv > 1024)
    return fail(B200FWD_EINVAL, name + ": the heads are a multiple of the kv heads, 1 to 1024 of them");
  if (hs < 16 || hs > 256 || hs % 16)
    return fail(B200FWD_EINVAL, name + ": the head size is a multiple of 16, at most 256");
  if ((int64_t)n * nh > INT32_MAX / 2 || n > 1 << 25)
    return fail(B200FWD_EINVAL, name + ": more rows (tokens times heads) than 2^30, or more tokens than 2^25");
  return 0;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200k_cache8_attention_scratch(int32_t n, int32_t n_seqs, int32_t nh, int32_t nkv, int32_t hs,
                                              int32_t half, uint64_t *bytes) {
  try {
    if (!bytes) return fail(B200FWD_EINVAL, "cache8_attention_scratch: null pointer");
    const int rc = check_sizes("cache8_attention_scratch", n, n_seqs, nh, nkv, hs);
    if (rc) return rc;
    *bytes = layout_of(n, n_seqs, nh, nkv, hs, half).bytes;
    return 0;
  } catch (...) {
    return fail(B200FWD_EINVAL, "cache8_attention_scratch: exception");
  }
}

extern "C" int b200k_cache8_attention_check(const void *scratch, b200fwd_stream stream) {
  try {
    if (!scratch || reinterpret_cast<uintptr_t>(scratch) % 256)
      return fail(B200FWD_EINVAL, "cache8_attention_check: scratch must be 256-byte aligned, and not null");
    int32_t code = 0;  // (Args::meta[-1].y)
    B200_CUDA(cudaMemcpyAsync(&code, reinterpret_cast<const int32_t *>(scratch) + 1, 4, cudaMemcpyDeviceToHost, as_stream(stream)));
    B200_CUDA(cudaStreamSynchronize(as_stream(stream)));
    if (code) return fail(B200FWD_ETIMEOUT, "cache8_attention: a pipeline wait gave up (code " + std::to_string(code) + ")");
    return 0;
  } catch (...) {
    return fail(B200FWD_EINVAL, "cache8_attention_check: exception");
  }
}

extern "C" int b200k_cache8_attention(void *out, const void *q, const int8_t *kc, const float *ks, const int8_t *vc,
                                      const float *vs, const int32_t *tables, const int32_t *starts,
                                      const int32_t *lengths, int32_t n, int32_t n_seqs, int32_t table_width,
                                      int32_t blocks, int32_t block, int32_t nh, int32_t nkv, int32_t hs,
                                      int64_t q_stride, int64_t out_stride, int32_t half, void *scratch,
                                      b200fwd_stream stream) {
  try {
    const char *what = "cache8_attention";
    int rc = check_sizes(what, n, n_seqs, nh, nkv, hs);
    if (!rc) rc = check_cache8(what, kc, ks, vc, vs, blocks, block, nkv, hs);
    if (rc) return rc;
    if (n == 0) return 0;
    if (!out || !q || !tables || !starts || !lengths || !scratch)
      return fail(B200FWD_EINVAL, "cache8_attention: null pointer");
    if (table_width < 1 || (int64_t)table_width * block > INT32_MAX / 2)
      return fail(B200FWD_EINVAL, "cache8_attention: a table row of 1 block at least and 2^30 positions at most");
    const int64_t row = (int64_t)nh * hs, to = half ? 8 : 4;
    if (q_stride < row || out_stride < row || q_stride % to || out_stride % to ||
        reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 16)
      return fail(B200FWD_EINVAL, "cache8_attention: rows of q and out of nh * hs values at least, on 16 bytes");
    if (reinterpret_cast<uintptr_t>(scratch) % 256)
      return fail(B200FWD_EINVAL, "cache8_attention: scratch must be 256-byte aligned");
    const Layout s = layout_of(n, n_seqs, nh, nkv, hs, half);
    uint8_t *base = reinterpret_cast<uint8_t *>(scratch);
    // blocks of tokens go to the tensor cores; where there is no more than a token a request on average (of the buffers'
    // rows), any request is taken here, and one kernel less launched
    const bool prompts = n > n_seqs && prompts_fit(hs);
    // Tables of no more positions than a span has: a thread block a tile, and nothing to join. No more requests than a block
    // looks over at once, as every block does (65,536 of them take 66 ms so). Measured, so and by spans: 3 requests of 333
    // positions 8.7 and 16.7 us, 64 of 512 23.7 and 28; 256 of 300 66 and 61.
    const bool whole_tiles = (int64_t)table_width * block <= MIN_UNITS * UNIT && n_seqs <= THREADS;
    Args a = {out, q, kc, vc, ks, vs, tables, starts, lengths, reinterpret_cast<int4 *>(base) + 1,
              reinterpret_cast<float2 *>(base + s.ml_at), reinterpret_cast<float *>(base + s.part_at), q_stride,
              out_stride, n, n_seqs, table_width, blocks, block, nkv, hs, nh / nkv,
              whole_tiles ? 1 : MIN_UNITS, whole_tiles, prompts ? ROWS_FEW : INT32_MAX,
              1.4426950408889634f / sqrtf((float)hs)};
    const cudaStream_t st = as_stream(stream);
    const int hseg = (hs + 63) / 64, blocks_x = (MOST_BLOCKS + nkv - 1) / nkv;
    const bool whole = hs % 64 == 0;
    const Launch launch_units = hseg == 1   ? launch_of<1>(s.rt, half, whole)
                                : hseg == 2 ? launch_of<2>(s.rt, half, whole)
                                : hseg == 3 ? launch_of<3>(s.rt, half, whole)
                                            : launch_of<4>(s.rt, half, whole);
    rc = launch_units(a, whole_tiles ? (int)(s.tiles < 65535 ? s.tiles : 65535) : blocks_x, st);
    if (!rc && prompts) rc = launch_attention8_prompts(a, half, st);
    if (rc || whole_tiles) return rc;
    return s.rt == 4   ? launch_combine<4, false>(a, s.tiles, st)
           : s.rt == 8 ? (half ? launch_combine<8, true>(a, s.tiles, st) : launch_combine<8, false>(a, s.tiles, st))
                       : (half ? launch_combine<16, true>(a, s.tiles, st) : launch_combine<16, false>(a, s.tiles, st));
  } catch (...) {
    return fail(B200FWD_EINVAL, "cache8_attention: exception");
  }
}
