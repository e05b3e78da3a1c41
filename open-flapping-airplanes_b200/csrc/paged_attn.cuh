// Attention of few rows over a paged cache: a token, or a few, per sequence, where reading the keys and values is all that counts.
//
// For each row: O = sum_j p_j v_j / sum_j p_j, p_j = 2^(s_j - m), s_j = scale log2(e) q.k_j, over the keys it sees, in one pass with a running
// maximum m. The rows of a key/value head (new tokens x the query heads that share it) are taken 8 or 16 at a time, as columns: S^T = K Q^T and O^T = V^T P^T are
// mma.sync products of 16 keys (or 16 head dims) by 8 rows, so that a single token of up to eight query heads wastes neither accumulators nor exponentials (with the rows as the
// 16 of a product a step of 32 keys took about 2,000 clocks and twice the registers). With few rows the
// tensor pipe idles whatever feeds it; what counts is bytes in flight, instructions per key and few steps between the last byte and the answer. A block's four warps take
// every fourth step of 16 or 32 keys and meet once, at the end; up to eight blocks that share the keys of a tile are a cluster and meet in shared memory, more leave their
// parts in the workspace for combine_kernel.
//
// Each warp has a ring of steps in shared memory. Where a page holds a multiple of 8 rows, boxes of 8 to 32 rows come through the copy engine, one instruction for
// 1 to 4 KB; other pages are gathered by cp.async, 16 bytes a lane. (Gathering everything kept the load/store pipe busy with the copies themselves: 29 clocks for
// 512 bytes, with the reads behind them, 4.8 TB/s over long contexts.) Rows lie 128 bytes wide, their 16-byte pieces permuted by the row number (the copy engine's
// swizzle), and operands are read in an order that meets no bank conflict; the order of the sum over head dims and the order of the output's dims are free as long as both
// operands agree:
//   scores   lane (r = lane / 4, c = lane % 4) reads of key r of 8 the pieces 2c and 2c + 1 of every 128 bytes; q is fetched in the same order
//   output   lane reads of keys 2c, 2c + 1, 2c + 8, 2c + 9 of 16 the piece r; two keys side by side make a word of the A operand, and rows r and r + 8
//            of the t-th product are two neighbouring dims
// The scores' accumulator has keys down the lanes, the second product wants them along a lane: movmatrix turns 8 x 8 of them.
//
// Rows of the 8-bit cache enter the products as bf16 of 2^-120 times their codes (paged::raw_pair, three instructions for two elements), which is exact, and so are the queries: bf16 as
// they came, a row's largest magnitude brought to 2^127 by a power of two. Keys' scales multiply the scores, values' scales the probabilities, which carry 2^100 so that nothing
// underflows (the result is 2^-20 of what it should be, made good at the end). Queries split into two e4m3 numbers against the keys as they are saved the widening, lost bits of elements
// below 2^-13 of a row's largest, and was no faster: 64 tokens over 4,096 keys, 32 heads over 8, 114 us against 112; four tokens each 160 against 144.
//
// A key that a row does not see counts nothing, whatever is stored there: its score is replaced, and where some rows of the tile see it and others do not,
// infinities and NaN are taken out of its values and added to the rows that see it. What lies behind the context in its last page may be fetched and counts nowhere; nothing
// of a bad page is read.
#pragma once
#include <cuda.h>
#include "paged.cuh"

namespace ofa {
namespace paged {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float RESCALE_LOG2 = 8.f;

struct AttnArgs {
  Batch b;
  Pool c;
  const bf16* q; long long q_row, q_head;
  bf16* out; long long o_row, o_head;
  float* lse;                       // [n_rows][n_heads] or null
  int n_heads, n_kv_heads, causal, window;
  Div group;
  float scale_log2;                 // of many_rows_kernel: its magnitude, flip = the scale is negative
  int flip, wide;                   // wide: offsets of 2^35 bytes and more
  alignas(64) CUtensorMap km, vm;   // the pages in boxes of `run` rows x 128 bytes (64: 8-bit rows of 64)
  int run;                          // a power of two, 8 .. 64 (few_rows_kernel: .. KEYS), or 0: pages of other sizes, no maps
  int tiles, nsplit;                // of the launch: row tiles per sequence (more are walked through), blocks that share a tile's keys
  int by_head, ranked;              // the order of blocks: in many_rows_kernel; sequences by length (at most 128)
  int cluster;                      // ... which are a cluster and meet in shared memory
  float* part;                      // otherwise, nsplit > 1: [row][head][split][D], and behind them float2 [row][head][split] = {m, l}
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ bool odd_bits(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }   // an infinity or a NaN in the pair
__device__ __forceinline__ uint32_t without_odd(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}

// A row's offset (a multiple of 16 bytes, -1: no row) from another lane: one exchange where the cache's offsets over 16 fit 31 bits
__device__ __forceinline__ long long from_lane(long long off, int lane, bool wide) {
  if (wide) return __shfl_sync(0xffffffffu, off, lane);
  const int v = __shfl_sync(0xffffffffu, (int)(off >> 4), lane);
  return v < 0 ? -1ll : (long long)v << 4;
}
// A bounded wait without a call (a function with an ABI of its own does not go with setmaxnreg). A try sleeps for about 300 clocks, the limit is a second or a few.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 10000000; i++) if (mbar_try(bar, parity)) return true;
  return false;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Shared memory of the cluster's other blocks. The barrier's instructions are for whole warps: their lanes come together first, from code that some of them had to themselves.
__device__ __forceinline__ void cluster_sync() { __syncwarp(); asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer(uint32_t addr, int rank) { uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank)); return r; }
__device__ __forceinline__ float peer_f32(uint32_t a) { float v; asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory"); return v; }
__device__ __forceinline__ float4 peer_f32x4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

// The sequence (of at most 128) with this place in their order by length, the longest first; scratch: 129 words of shared memory. For all threads of a block of 128 or more.
__device__ __forceinline__ int by_length(const Batch& B, int place, int* scratch) {
  const int t = threadIdx.x, len = t < B.n_seqs ? __ldg(B.kv_len + t) : -1;
  if (t < 128) scratch[t] = len;
  __syncthreads();
  if (t < B.n_seqs) {
    int rank = 0;
    for (int j = 0; j < B.n_seqs; j++) rank += scratch[j] > len || (scratch[j] == len && j < t);
    if (rank == place) scratch[128] = t;
  }
  __syncthreads();
  return scratch[128];
}

// The first key that a row at position pos sees; without a difference that leaves 32 bits (positions may be negative, and windows as large as an int)
__device__ __forceinline__ int first_seen(const AttnArgs& P, int pos) { return P.window && pos >= P.window ? pos - P.window + 1 : 0; }
// Whether a row at position pos of sequence i sees any key. Asked only where the sum of a row's exponentials is 0: a row that sees nothing gets zeros, one whose scores are all
// -inf has no softmax, and gets NaN.
__device__ __forceinline__ bool sees_any(const AttnArgs& P, int i, int pos) {
  const int cap = reach(P.b, __ldg(P.b.kv_len + i)), hi = P.causal ? min(cap, pos + 1) : cap, lo = first_seen(P, pos);
  if (hi <= lo) return false;
  const unsigned last = P.b.page.quot((unsigned)(hi - 1));
#pragma unroll 1
  for (unsigned idx = P.b.page.quot((unsigned)lo); idx <= last; idx++)
    if ((unsigned)__ldg(P.b.pages + (long long)i * P.b.pages_stride + idx) < (unsigned)P.b.n_pages) return true;
  return false;
}
// What a row's sums are multiplied by, for l the sum of its exponentials
__device__ __forceinline__ float over(const AttnArgs& P, float l, int i, int pos) { return l != 0.f ? 1.f / l : sees_any(P, i, pos) ? __int_as_float(0x7fc00000) : 0.f; }

template <int D, bool E4M3, int NR> struct Few {
  static constexpr int RB = D * (E4M3 ? 1 : 2);                 // bytes of a row
  static constexpr int KEYS = RB > 128 ? 16 : 32, WARPS = 4, ROWS = 8 * NR;      // of a step: at most 8 KB of keys and values a warp
  static constexpr int NB = KEYS / 16;
  static constexpr int W = RB > 128 ? 128 : RB, HALVES = RB / W;                 // rows lie W bytes wide, in one or two parts
  static constexpr int KP = RB / 64;                            // 16-byte pieces of a key that a lane reads
  static constexpr int VB = RB / 8, VW = VB >= 16 ? 16 : 8, VP = VB / VW;        // bytes of a value row that a lane reads, in pieces of VW
  static constexpr int TILE = KEYS * RB, STAGE = 2 * TILE;      // K, then V
  static constexpr int STAGES = STAGE >= 8192 ? 2 : 3;
  static constexpr uint32_t ALL = KEYS == 32 ? 0xffffffffu : 0xffffu;
  static constexpr int PAD = D + 8;                             // floats of a row where the warps meet
  static constexpr int BARS_AT = WARPS * STAGES * STAGE, SMEM = BARS_AT + WARPS * STAGES * 8 + 1024;      // 1,024 for the alignment of the swizzle's atoms
  static_assert(WARPS * ROWS * (PAD + 2) * 4 <= BARS_AT, "the meeting of the warps does not fit");
  // where piece `chunk` (16 bytes) of a row lies
  static __device__ __forceinline__ uint32_t at(int row, int chunk) {
    if constexpr (W == 64) return (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
    else return (uint32_t)((chunk >> 3) * (KEYS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
  }
};

// one held element as a float (the rare path)
template <bool E4M3> __device__ float held(const char* row, int d, int scale) {
  if constexpr (E4M3) return __uint_as_float(widen_lo(*reinterpret_cast<const unsigned char*>(row + d), scale_bits(scale)) << 16);
  return to_f(reinterpret_cast<const bf16*>(row)[d]);
}

template <int D, bool E4M3, int NR>
__global__ void __launch_bounds__(128, NR == 1 ? 3 : 2) few_rows_kernel(const __grid_constant__ AttnArgs P) {
  using F = Few<D, E4M3, NR>;
  constexpr int MT = D / 16, KS = E4M3 ? D / 32 : D / 16;        // products of 16 dims of the output; of 16 (32: 8-bit keys) dims of a score
  extern __shared__ __align__(16) unsigned char raw[];
  unsigned char* smem = raw + (-(int)smem_u32(raw) & 1023);      // by an offset: through an integer the pointer would lose its address space
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const uint32_t bars = smem_u32(smem + F::BARS_AT) + warp * F::STAGES * 8;
  if (lane < F::STAGES) mbar_init(bars + lane * 8, 1);
  mbar_fence_init();
  __syncwarp();
  after_the_kernel_before();
  uint32_t used = 0;                                             // steps of this warp so far: phases of its barriers
  const int split = (int)blockIdx.x % P.nsplit, rest = (int)blockIdx.x / P.nsplit, kvh = rest % P.n_kv_heads, tile0 = rest / P.n_kv_heads % P.tiles;
  int seq = rest / P.n_kv_heads / P.tiles;
  if (P.ranked) {
    seq = by_length(P.b, seq, reinterpret_cast<int*>(smem));     // where the rings will be
    fence_async_shared();                                        // read, before the copy engine writes there
    __syncthreads();
  }
  const Chunk ch = chunk_of(P.b, seq);
  const int group = (int)P.group.d, cap = reach(P.b, ch.len);
  if (ch.len > cap && threadIdx.x == 0) flag(P.b.status, ST_LENGTH);
  unsigned char* ring = smem + warp * F::STAGES * F::STAGE;
  const uint32_t ring_s = smem_u32(ring);
  const char* kb = P.c.k + (long long)kvh * P.c.head_b;
  const char* vb = P.c.v + (long long)kvh * P.c.head_b;
  // where this lane's pieces lie in a tile: keys' rows r, values' rows 2c and 2c + 1; rows 8 further are 8 W bytes further
  const uint32_t ka0 = F::at(r, F::W == 64 ? c : 2 * c), ka1 = F::W == 64 ? ka0 : F::at(r, 2 * c + 1);
  const uint32_t va0 = F::at(2 * c, F::W == 64 ? r >> 1 : r) + (F::VW == 8 ? (r & 1) * 8 : 0), va1 = F::at(2 * c + 1, F::W == 64 ? r >> 1 : r) + (F::VW == 8 ? (r & 1) * 8 : 0);
  // the dim of row r (or r + 8: the one behind it) in the t-th product of the output
  auto dim_of = [&](int t) { return E4M3 ? r * (D / 8) + 2 * t : (t / 4) * 64 + r * 8 + (t % 4) * 2; };

  for (int tile = tile0; tile * F::ROWS < ch.n * group; tile += P.tiles) {
    const int t_last = min(ch.n - 1, (int)P.group.quot(tile * F::ROWS + F::ROWS - 1)), p_min = ch.p0 + (int)P.group.quot(tile * F::ROWS), p_max = ch.p0 + t_last;
    uint32_t qf[NR][D / 16][2];                                  // row r of every eight
    float rowf[NR][2];                                           // what the raw scores of rows 2c and 2c + 1 of every eight are multiplied by
    int pos[NR][2];                                              // and where they stand
#pragma unroll
    for (int n = 0; n < NR; n++) {
      const int rr = tile * F::ROWS + n * 8 + r, t = (int)P.group.quot(rr);
      const bool on = t < ch.n;
      const bf16* src = P.q + (long long)(on ? ch.s + t : ch.s) * P.q_row + (long long)(kvh * group + rr - t * group) * P.q_head;
      uint4 qv[E4M3 ? KS : 1];
#pragma unroll
      for (int s = 0; s < KS; s++) {
        if constexpr (E4M3) qv[s] = on ? *reinterpret_cast<const uint4*>(src + (D == 128 ? (2 * c + s / 2) * 16 : c * 16) + s % 2 * 8) : make_uint4(0, 0, 0, 0);
        else {
          const uint2 w = on ? *reinterpret_cast<const uint2*>(src + (s / 4) * 64 + (2 * c + s / 2 % 2) * 8 + s % 2 * 4) : make_uint2(0, 0);
          qf[n][s][0] = w.x; qf[n][s][1] = w.y;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int t2 = (int)P.group.quot(tile * F::ROWS + n * 8 + 2 * c + h);
        pos[n][h] = t2 < ch.n ? ch.p0 + t2 : p_max;
        rowf[n][h] = P.scale_log2;
      }
      if constexpr (E4M3) {                                      // the row's largest magnitude to 2^127, since widened keys are 2^-120 of theirs
        unsigned mag = 0;
#pragma unroll
        for (int s = 0; s < KS; s++) mag = max(mag, max_bits(qv[s]));
        mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
        mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 2));
        const int shift = min(max(127 - ((int)(mag >> 7) - 127), 0), 127);
        const float up = __uint_as_float((uint32_t)(127 + shift) << 23), down = __uint_as_float((uint32_t)(247 - shift) << 23);      // 2^(120 - shift)
        auto times_up = [&](uint32_t w) { const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)); return pack2f(x.x * up, x.y * up); };
#pragma unroll
        for (int s = 0; s < KS; s++) { qf[n][2 * s][0] = times_up(qv[s].x); qf[n][2 * s][1] = times_up(qv[s].y); qf[n][2 * s + 1][0] = times_up(qv[s].z); qf[n][2 * s + 1][1] = times_up(qv[s].w); }
#pragma unroll
        for (int h = 0; h < 2; h++) rowf[n][h] *= __shfl_sync(0xffffffffu, down, (2 * c + h) * 4);
      }
    }
    const int hi = min(cap, P.causal ? p_max + 1 : ch.len), lo = first_seen(P, p_min);
    const int first = lo / F::KEYS, nst = max(0, (hi + F::KEYS - 1) / F::KEYS - first);
    const int a = first + (int)((long long)nst * split / P.nsplit) + warp, b = first + (int)((long long)nst * (split + 1) / P.nsplit);
    const int mine = b > a ? (b - a + F::WARPS - 1) / F::WARPS : 0;

    float o[NR][MT][4], m[NR][2], l[NR][2];
#pragma unroll
    for (int n = 0; n < NR; n++) {
      m[n][0] = m[n][1] = -INFINITY; l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int t = 0; t < MT; t++) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.f;
    }

    // the page of this lane's key in the warp's i-th step (of its run of keys, as far as the tile reaches into it); asked for a step ahead
    const int run = P.run ? P.run : 1;
    auto page_of = [&](int i) {
      const int p = (a + i * F::WARPS) * F::KEYS + (lane & (F::KEYS - 1));
      if (i >= mine || (p | (run - 1)) < lo || (p & -run) >= hi) return -1;
      return __ldg(P.b.pages + (long long)seq * P.b.pages_stride + P.b.page.quot((unsigned)(p & -run)));      // below cap: within the table
    };
    int page = page_of(0);
    uint32_t keys[F::STAGES], ks8[F::STAGES], vs8[F::STAGES];    // of the steps on their way, the last one first: which keys are there, scale bytes of this lane's
    auto issue = [&](int i) {                                    // the warp's i-th step
#pragma unroll
      for (int x = F::STAGES - 1; x > 0; x--) { keys[x] = keys[x - 1]; ks8[x] = ks8[x - 1]; vs8[x] = vs8[x - 1]; }
      if (i >= mine) return;
      const int p = (a + i * F::WARPS) * F::KEYS + (lane & (F::KEYS - 1));
      const int at = p - (int)(P.b.page.quot((unsigned)p) * P.b.page.d), pg = page;
      const bool inside = p >= lo && p < hi, there = (unsigned)pg < (unsigned)P.b.n_pages, ok = inside && there;
      if (inside && !there) flag(P.b.status, ST_PAGE);
      page = page_of(i + 1);
      keys[0] = __ballot_sync(0xffffffffu, ok) & F::ALL;
      if constexpr (E4M3) {
        const long long so = (long long)pg * P.c.s_page + (long long)kvh * P.c.s_head + (long long)at * P.c.s_row;
        ks8[0] = ok ? __ldg(P.c.ks + so) : 127; vs8[0] = ok ? __ldg(P.c.vs + so) : 127;
      }
      const uint32_t slot = (used + (uint32_t)i) % F::STAGES, dk = ring_s + slot * F::STAGE, dv = dk + F::TILE;
      if (P.run) {                                               // the first lane of a run asks for its boxes
        const bool first_of = there && lane < F::KEYS && (lane & (run - 1)) == 0;
        const uint32_t bar = bars + slot * 8, n = __popc(__ballot_sync(0xffffffffu, first_of));
        if (lane == 0) mbar_expect_tx(bar, n * (uint32_t)(run * F::RB * 2));
        __syncwarp();
        if (first_of) {
#pragma unroll
          for (int h = 0; h < F::HALVES; h++) {
            tma_load_4d(dk + h * (F::KEYS * 128) + lane * F::W, &P.km, bar, h * 64, at, kvh, pg);
            tma_load_4d(dv + h * (F::KEYS * 128) + lane * F::W, &P.vm, bar, h * 64, at, kvh, pg);
          }
        }
      } else {
        constexpr int CH = F::RB / 16, N = F::KEYS * CH / 32;
        const long long off = ok ? (long long)pg * P.c.page_b + (long long)at * P.c.row_b : -1;
        long long o[N];                                          // all the exchanges before the first copy: in turns each copy would wait for its own
#pragma unroll
        for (int x = 0; x < N; x++) o[x] = from_lane(off, (x * 32 + lane) / CH, P.wide);
#pragma unroll
        for (int x = 0; x < N; x++) {
          const bool on = o[x] >= 0;
          const long long src = (on ? o[x] : 0) + lane % CH * 16;
          const uint32_t to = F::at((x * 32 + lane) / CH, lane % CH);
          cp16(dk + to, kb + src, on);
          cp16(dv + to, vb + src, on);
        }
      }
    };
    bool fine = true;
    auto step = [&](int i) {
      const uint32_t slot = (used + (uint32_t)i) % F::STAGES;
      const int k0 = (a + i * F::WARPS) * F::KEYS;
      unsigned char* sk = ring + slot * F::STAGE;
      unsigned char* sv = sk + F::TILE;
      if (P.run) { if (!wait_for(bars + slot * 8, ((used + (uint32_t)i) / F::STAGES) & 1)) fine = false; }
      else { cp_wait<F::STAGES - 1>(); __syncwarp(); }
      const uint32_t valid = keys[F::STAGES - 1];
      float kf = 1.f, vf = 1.f;                                  // of this lane's key: its scale, 2^100 times its values' scale
      if constexpr (E4M3) {
        const int k8 = (int)ks8[F::STAGES - 1], v8 = (int)vs8[F::STAGES - 1];
        kf = __uint_as_float(k8 == SCALE_NAN ? 0x7fc00000u : (uint32_t)min(max(k8, 1), E_MAX + 127) << 23);
        vf = __uint_as_float(v8 == SCALE_NAN ? 0x7fc00000u : (uint32_t)(min(v8, E_MAX + 127) + 100) << 23);
      }
      const bool mask = valid != F::ALL || (P.causal && k0 + F::KEYS - 1 > p_min) || (P.window && k0 < first_seen(P, p_max));
      float s[F::NB][NR][4];
      float fk[F::NB][2], fv[F::NB][2];
#pragma unroll
      for (int kk = 0; kk < F::NB; kk++) {
#pragma unroll
        for (int n = 0; n < NR; n++) s[kk][n][0] = s[kk][n][1] = s[kk][n][2] = s[kk][n][3] = 0.f;
        float s2[NR][4] = {};                                    // two chains of products
        if constexpr (E4M3) {
#pragma unroll
          for (int h = 0; h < 2; h++) { fk[kk][h] = __shfl_sync(0xffffffffu, kf, kk * 16 + h * 8 + r); fv[kk][h] = __shfl_sync(0xffffffffu, vf, kk * 16 + h * 8 + r); }
        }
#pragma unroll
        for (int x = 0; x < F::KP; x++) {
          const unsigned char* src = sk + (x & 1 ? ka1 : ka0) + x / 2 * (F::KEYS * 128) + kk * 16 * F::W;
          const uint4 wa = *reinterpret_cast<const uint4*>(src), wb = *reinterpret_cast<const uint4*>(src + 8 * F::W);
          if constexpr (E4M3) {
            const uint32_t ua[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t a0[4] = {raw_pair(ua[i], ua[i], raw_sel(0, 1)), raw_pair(ub[i], ub[i], raw_sel(0, 1)), raw_pair(ua[i], ua[i], raw_sel(2, 3)), raw_pair(ub[i], ub[i], raw_sel(2, 3))};
#pragma unroll
              for (int n = 0; n < NR; n++) mma16816(i % 2 ? s2[n] : s[kk][n], a0, qf[n][4 * x + i][0], qf[n][4 * x + i][1]);
            }
          } else {
            const uint32_t a0[4] = {wa.x, wb.x, wa.y, wb.y}, a1[4] = {wa.z, wb.z, wa.w, wb.w};
#pragma unroll
            for (int n = 0; n < NR; n++) {
              mma16816(s[kk][n], a0, qf[n][2 * x][0], qf[n][2 * x][1]);
              mma16816(s2[n], a1, qf[n][2 * x + 1][0], qf[n][2 * x + 1][1]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[kk][n][e] += s2[n][e];
      }
      float mx[NR][2];
#pragma unroll
      for (int n = 0; n < NR; n++) {
        mx[n][0] = mx[n][1] = -INFINITY;
#pragma unroll
        for (int kk = 0; kk < F::NB; kk++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float& x = s[kk][n][e];
            x *= E4M3 ? rowf[n][e & 1] * fk[kk][e >> 1] : rowf[n][e & 1];      // a key's scale is a power of two: first with the row's factor, a large query's sum may not have room for it
            if (mask) {
              const int at = kk * 16 + (e >> 1) * 8 + r, p = k0 + at, q = pos[n][e & 1];
              if (!((valid >> at) & 1) || (P.causal && p > q) || (P.window && p < first_seen(P, q))) x = -INFINITY;
            }
            mx[n][e & 1] = fmaxf(mx[n][e & 1], x);
          }
      }
      // The reference that a row's exponentials are taken against is raised only when some score has passed it by 2^8 (they stay below 256, exact enough in fp32 sums and
      // bf16): in most steps one vote replaces the search of the maximum over the lanes.
      bool up = false;
#pragma unroll
      for (int n = 0; n < NR; n++) up |= mx[n][0] > m[n][0] + RESCALE_LOG2 || mx[n][1] > m[n][1] + RESCALE_LOG2;
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int n = 0; n < NR; n++) {
          float al[2];
#pragma unroll
          for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx[n][h] = fmaxf(mx[n][h], __shfl_xor_sync(0xffffffffu, mx[n][h], d));
            const float mn = fmaxf(m[n][h], mx[n][h]);
            al[h] = mn == -INFINITY ? 1.f : ex2_approx(m[n][h] - mn);
            m[n][h] = mn; l[n][h] *= al[h];
          }
#pragma unroll
          for (int t = 0; t < MT; t++) { o[n][t][0] *= al[0]; o[n][t][1] *= al[1]; o[n][t][2] *= al[0]; o[n][t][3] *= al[1]; }
        }
      }
      if (mask) {                                                // values that some row must not meet: none of them may be an infinity or a NaN
        bool odd = false;
        if constexpr (E4M3) {
          odd = vf != vf && ((valid >> (lane & (F::KEYS - 1))) & 1);
#pragma unroll
          for (int kk = 0; kk < F::NB; kk++)
#pragma unroll
            for (int h = 0; h < 2; h++) if (fv[kk][h] != fv[kk][h]) fv[kk][h] = 0.f;
        } else {
#pragma unroll 1
          for (int x = 0; x < F::TILE / 512; x++) {
            uint4* w = reinterpret_cast<uint4*>(sv + x * 512 + lane * 16);
            uint4 u = *w;
            if (odd_bits(u.x) || odd_bits(u.y) || odd_bits(u.z) || odd_bits(u.w)) {
              odd |= valid >> ((x * 512 + lane * 16) / F::W % F::KEYS) & 1;
              *w = make_uint4(without_odd(u.x), without_odd(u.y), without_odd(u.z), without_odd(u.w));
            }
          }
        }
        if constexpr (!E4M3) {
          fence_async_shared();                                  // what was taken out, before the copy engine writes there again
          __syncwarp();
        }
        if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
          for (int kk = 0; kk < F::KEYS; kk++) {
            const int p = k0 + kk;
            int page, at;
            if (!((valid >> kk) & 1) || !locate(P.b, seq, p, page, at)) continue;
            const char* row = vb + (long long)page * P.c.page_b + (long long)at * P.c.row_b;
            const int sc = E4M3 ? P.c.vs[(long long)page * P.c.s_page + (long long)kvh * P.c.s_head + (long long)at * P.c.s_row] : 0;
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const float x = held<E4M3>(row, dim_of(t) + e, sc);
                if (isfinite(x)) continue;
#pragma unroll
                for (int n = 0; n < NR; n++)
#pragma unroll
                  for (int h = 0; h < 2; h++) if (!(P.causal && p > pos[n][h]) && p >= first_seen(P, pos[n][h])) o[n][t][2 * e + h] += x;
              }
          }
          __syncwarp();                                          // the products below are whole warps' too
        }
      }
#pragma unroll
      for (int kk = 0; kk < F::NB; kk++) {
        uint32_t pf[NR][2];                                      // P^T: rounded to bf16 for the product (half a step, 2^-8 of each term); the sum l is taken before
#pragma unroll
        for (int n = 0; n < NR; n++) {
          const float m0 = m[n][0] == -INFINITY ? 0.f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.f : m[n][1];      // a row that has seen no key yet: 2^(-inf - 0) = 0
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float p0 = ex2_approx(s[kk][n][2 * h] - m0), p1 = ex2_approx(s[kk][n][2 * h + 1] - m1);
            l[n][0] += p0; l[n][1] += p1;
            if constexpr (E4M3) { p0 *= fv[kk][h]; p1 *= fv[kk][h]; }
            asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pf[n][h]) : "r"(pack2f(p0, p1)));
          }
        }
#pragma unroll
        for (int x = 0; x < F::VP; x++) {
          uint32_t w[4][F::VW / 4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const unsigned char* src = sv + (j & 1 ? va1 : va0) + x * (F::KEYS * 128) + (kk * 16 + (j >> 1) * 8) * F::W;
            if constexpr (F::VW == 16) {
              const uint4 u = *reinterpret_cast<const uint4*>(src);
              w[j][0] = u.x; w[j][1] = u.y; w[j][2] = u.z; w[j][3] = u.w;
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(src);
              w[j][0] = u.x; w[j][1] = u.y;
            }
          }
          constexpr int TP = E4M3 ? F::VW / 2 : 4;               // products of a piece
#pragma unroll
          for (int t = 0; t < TP; t++) {
            uint32_t af[4];
            if constexpr (E4M3) {                                // bytes 2t and 2t + 1 of a piece, of two keys each
              const int y = t / 2, z = (t % 2) * 2;
              af[0] = raw_pair(w[0][y], w[1][y], raw_sel(z, 4 + z)); af[1] = raw_pair(w[0][y], w[1][y], raw_sel(z + 1, 5 + z));
              af[2] = raw_pair(w[2][y], w[3][y], raw_sel(z, 4 + z)); af[3] = raw_pair(w[2][y], w[3][y], raw_sel(z + 1, 5 + z));
            } else {
              af[0] = __byte_perm(w[0][t], w[1][t], 0x5410); af[1] = __byte_perm(w[0][t], w[1][t], 0x7632);
              af[2] = __byte_perm(w[2][t], w[3][t], 0x5410); af[3] = __byte_perm(w[2][t], w[3][t], 0x7632);
            }
#pragma unroll
            for (int n = 0; n < NR; n++) mma16816(o[n][x * TP + t], af, pf[n][0], pf[n][1]);
          }
        }
      }
    };

    // One copy of each part of the code: a short context runs through it once, fetching it from L2
#pragma unroll 1
    for (int i = 0; i < mine + F::STAGES - 1; i++) {
      issue(i);
      if (!P.run) cp_commit();
      if (i >= F::STAGES - 1) step(i - (F::STAGES - 1));
      __syncwarp();                                              // all lanes have read what the next copies overwrite
    }
    used += (uint32_t)mine;
    if (!fine) flag(P.b.status, ST_TIMEOUT);
    cp_wait<0>();
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], d);

    // the warps meet: rows of D sums each, and {m, l}
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);
    float2* sm = reinterpret_cast<float2*>(so + F::WARPS * F::ROWS * F::PAD);
    constexpr float MEND = E4M3 ? 1048576.f : 1.f;               // 2^20
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = warp * F::ROWS + n * 8 + 2 * c + h;
#pragma unroll
        for (int t = 0; t < MT; t++) *reinterpret_cast<float2*>(so + row * F::PAD + dim_of(t)) = make_float2(o[n][t][h] * MEND, o[n][t][2 + h] * MEND);
        if (r == 0) sm[row] = make_float2(m[n][h], l[n][h]);
      }
    __syncthreads();
    {
      constexpr int TPR = 128 / F::ROWS, DP = D / TPR;           // threads a row, dims a thread: a thread's are 4 side by side in every 4 * TPR
      const int row = threadIdx.x / TPR, part = threadIdx.x % TPR, rr = tile * F::ROWS + row, t = (int)P.group.quot(rr);
      float mm = -INFINITY, ll = 0.f, acc[DP] = {};
#pragma unroll
      for (int w = 0; w < F::WARPS; w++) mm = fmaxf(mm, sm[w * F::ROWS + row].x);
#pragma unroll
      for (int w = 0; w < F::WARPS; w++) {
        const float2 ml = sm[w * F::ROWS + row];
        const float f = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - mm);      // no key seen, or only scores of -inf: sums of 0, or not finite
        ll += ml.y * f;
#pragma unroll
        for (int x = 0; x < DP; x += 4) {
          const float4 v = *reinterpret_cast<const float4*>(so + (w * F::ROWS + row) * F::PAD + x * TPR + part * 4);
          acc[x] += v.x * f; acc[x + 1] += v.y * f; acc[x + 2] += v.z * f; acc[x + 3] += v.w * f;
        }
      }
      const int head = kvh * group + rr - t * group;
      const long long g = (long long)(ch.s + t) * P.n_heads + head;
      bool last = t < ch.n;                                      // this thread writes the row's result
      if (P.cluster) {                                           // the blocks of the cluster meet in each other's shared memory, rows dealt out among them
        __syncthreads();
#pragma unroll
        for (int x = 0; x < DP; x += 4) *reinterpret_cast<float4*>(so + row * F::PAD + x * TPR + part * 4) = make_float4(acc[x], acc[x + 1], acc[x + 2], acc[x + 3]);
        if (part == 0) sm[row] = make_float2(mm, ll);
        cluster_sync();
        last = last && row % P.nsplit == split;
        if (last) {
          const uint32_t at = smem_u32(so + row * F::PAD + part * 4), am = smem_u32(sm + row);
          mm = -INFINITY; ll = 0.f;
          for (int s = 0; s < P.nsplit; s++) mm = fmaxf(mm, peer_f32(peer(am, s)));
#pragma unroll
          for (int x = 0; x < DP; x++) acc[x] = 0.f;
          for (int s = 0; s < P.nsplit; s++) {
            const float m1 = peer_f32(peer(am, s)), f = m1 == -INFINITY ? 1.f : ex2_approx(m1 - mm);
            ll += peer_f32(peer(am, s) + 4) * f;
            const uint32_t src = peer(at, s);
#pragma unroll
            for (int x = 0; x < DP; x += 4) {
              const float4 v = peer_f32x4(src + x * TPR * 4);
              acc[x] += v.x * f; acc[x + 1] += v.y * f; acc[x + 2] += v.z * f; acc[x + 3] += v.w * f;
            }
          }
        }
      }
      if (last && (P.cluster || P.nsplit == 1)) {
        const float inv = over(P, ll, seq, ch.p0 + t);
        bf16* dst = P.out + (long long)(ch.s + t) * P.o_row + (long long)head * P.o_head + part * 4;
#pragma unroll
        for (int x = 0; x < DP; x += 4) *reinterpret_cast<uint2*>(dst + x * TPR) = make_uint2(pack2f(acc[x] * inv, acc[x + 1] * inv), pack2f(acc[x + 2] * inv, acc[x + 3] * inv));
        if (P.lse && part == 0) P.lse[g] = ll == 0.f ? -INFINITY : mm * LN2 + logf(ll);
      } else if (last) {
        float* dst = P.part + (g * P.nsplit + split) * D + part * 4;
#pragma unroll
        for (int x = 0; x < DP; x += 4) *reinterpret_cast<float4*>(dst + x * TPR) = make_float4(acc[x], acc[x + 1], acc[x + 2], acc[x + 3]);
        if (part == 0) reinterpret_cast<float2*>(P.part + (long long)P.b.n_rows * P.n_heads * P.nsplit * D)[g * P.nsplit + split] = make_float2(mm, ll);
      }
      if (P.cluster) cluster_sync();                             // nobody's shared memory goes while another reads it
    }
    fence_async_shared();
    __syncthreads();
  }
}

// Joins the splits (at most 64) of a row and head, in their order: a warp each. Rows that no sequence brings, or one that chunk_of leaves out, have no parts and are left as they are: the
// warp looks for the row's sequence by chunk_of's rule (32 at once; calls whose keys are split into parts have few sequences).
template <int D> __global__ void __launch_bounds__(128) combine_kernel(const __grid_constant__ AttnArgs P) {
  const long long g = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int row = (int)(g / P.n_heads), head = (int)(g - (long long)row * P.n_heads);
  int seq = -1;
  for (int i0 = 0; i0 < P.b.n_seqs && seq < 0; i0 += 32) {
    const int i = min(i0 + lane, P.b.n_seqs - 1), s = __ldg(P.b.q_start + i), e = __ldg(P.b.q_start + i + 1);
    const uint32_t here = __ballot_sync(0xffffffffu, s >= 0 && e <= P.b.n_rows && s <= row && row < e);
    if (here) seq = min(i0 + __ffs(here) - 1, P.b.n_seqs - 1);
  }
  cudaGridDependencySynchronize();
  if (seq < 0) return;
  const float2* ml = reinterpret_cast<const float2*>(P.part + (long long)P.b.n_rows * P.n_heads * P.nsplit * D) + g * P.nsplit;
  float2 a = lane < P.nsplit ? ml[lane] : make_float2(-INFINITY, 0.f), b = lane + 32 < P.nsplit ? ml[lane + 32] : make_float2(-INFINITY, 0.f);
  const float mm = warp_max(fmaxf(a.x, b.x));
  const float fa = a.x == -INFINITY ? 1.f : ex2_approx(a.x - mm), fb = b.x == -INFINITY ? 1.f : ex2_approx(b.x - mm);
  const float ll = warp_sum(a.y * fa + b.y * fb);
  constexpr int DP = D / 32;
  float acc[DP] = {};
  const float* src = P.part + g * P.nsplit * D + lane * DP;
  for (int s = 0; s < P.nsplit; s++) {
    const float f = __shfl_sync(0xffffffffu, s < 32 ? fa : fb, s & 31);
#pragma unroll
    for (int x = 0; x < DP; x++) acc[x] += src[(long long)s * D + x] * f;
  }
  const float inv = over(P, ll, seq, __ldg(P.b.kv_len + seq) - __ldg(P.b.q_start + seq + 1) + row);
  bf16* dst = P.out + (long long)row * P.o_row + (long long)head * P.o_head + lane * DP;
#pragma unroll
  for (int x = 0; x < DP; x += 2) *reinterpret_cast<uint32_t*>(dst + x) = pack2f(acc[x] * inv, acc[x + 1] * inv);
  if (P.lse && lane == 0) P.lse[g] = ll == 0.f ? -INFINITY : mm * LN2 + logf(ll);
}

}  // namespace paged
}  // namespace ofa
