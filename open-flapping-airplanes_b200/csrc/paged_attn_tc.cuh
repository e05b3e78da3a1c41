// Attention of many rows over a paged cache on the 5th-generation tensor cores: chunks of new tokens, where the products count.
//
// The rows of a key/value head (new tokens x the query heads that share it) are taken 128 at a time, a tile, and walk their keys 128 at a time. A block has two tiles, half
// a step apart, so that the tensor pipe works for one while the softmax warps of the other do; heads of 64 with bf16 rows, whose tiles are small, have one tile a block and two blocks
// an SM, which also covers a block's start and end (four prompts of 1,024 tokens, 12 heads: 32.1 -> 29.0 us). So have up to 64 rows of heads of 128 (drafts): their tile is 64 rows high, and warps
// without rows only pass their signals on (5 tokens of 24 sequences over up to 2,000 keys, 32 heads over 8: 54.4 -> 41.2 us; of 64 sequences over 4,096: 236 -> 176, 6.1 TB/s; with two
// tiles of keys and values instead of three on an SM's half 55 and 204). A block's start and end take 6 us, most of it instructions that are fetched for the first time: they are kept short, in rolled loops. Roles of a block's warps:
//   softmax    four warps a tile, a thread per row (= tensor-memory lane): reads its 128 scores once, keeps maximum and sum, writes the probabilities
//              back over the second half of them as bf16, the A operand of the second product
//   products   a warp a tile, one thread of which issues, in halves of 64 keys so that little of a step waits for all of the one before: the first half of the next scores as
//              soon as the present ones are in registers, O += P V of each half when its probabilities are written, then the second half of the next scores. (4,096 tokens over
//              16,384 keys, heads of 128: 843 us, 860 now; without the early half 1,075. Steps of 64 keys with two buffers of scores waited least, but their fixed cost of 420 clocks came twice: 928;
//              two threads a row, four softmax warps a scheduler: 910, bound by issue; a third of the exponentials by a polynomial on the multiply-add pipe: 970 and more, for registers and issue.)
//              One thread a tile because one issues a tcgen05.mma only every ~96 clocks and a 128 x 128 x 16 product takes 64
//   copies     one warp asks the copy engine for keys and values, in boxes of 8 to 64 rows of a page: bf16 rows into a ring of tiles in the layout the products read
//              (128-byte swizzle), 8-bit rows into a ring of their own
//   workers    widen 8-bit rows from there into the tiles, once for the block's rows, a worker on each scheduler; look at values that some row must not meet; and gather the rows of pages that are no
//              multiple of 8 by cp.async, 16 bytes a lane
// What bounds it: 128 keys of two tiles of heads of 128 take 3,400 clocks, of which the tensor pipe works 2,048 and the special-function unit, for 32,768 exponentials, as many.
// Tensor memory: S of a tile in 128 columns (P in their last 64), O behind all S.
//
// A row's probabilities are taken against a reference that is raised only when the true maximum has passed it by 2^8 (they stay below 256: exact enough in fp32 sums and
// bf16), and only then is the row of O multiplied in tensor memory. A step's scores are complete only when the product before them is, since one thread's products run in their order: a softmax thread
// that has its scores may also rewrite its row of O.
//
// Keys that some rows of the block see and others do not (the diagonal, the window's edge, the end of the context) come in tiles whose values are all looked
// at: infinities and NaN are taken out and added at the end to the rows that see them.
#pragma once
#include "attn_tc.cuh"
#include "paged_attn.cuh"

namespace ofa {
namespace paged {

template <int D, bool E4M3, int NT> struct Tc {                 // NT tiles of 128 rows a block
  static constexpr int BLOCKS = E4M3 ? 1 : 3 - NT;              // of an SM
  // Rows of a tile that are used: 64 where two blocks of wide rows share an SM. Q's parts then lie 64 rows apart, which leaves room for a third tile of keys or values (products read
  // the other 64 rows from whatever lies behind, and nobody looks at what comes of them)
  static constexpr int ROWS = NT == 1 && D == 128 ? 64 : 128, Q_PART = ROWS * 128, Q_TILE = ROWS * D * 2;
  // 8-bit rows: one or two workers on each scheduler, the rest idle
  static constexpr int WORKERS = E4M3 ? (NT == 1 ? 8 : 4) : NT == 1 ? 2 : 5, WARPS = BLOCKS == 2 ? 8 : 16, THREADS = 32 * WARPS;
  static constexpr int SOFT_REGS = 184, REST_REGS = 72;         // of a softmax thread, of another: together twice the launch's 128
  static constexpr int TMEM = NT * 256, O_AT = NT * 128;        // columns; S of a tile at tile * 128, O behind them
  static constexpr int TILE = 128 * D * 2;                      // a tile of rows: D / 64 parts of 128 rows x 128 bytes
  static constexpr int NST = E4M3 ? (D == 64 ? 6 : 5 - NT) : NT == 1 && D == 128 ? 3 : 4;           // ring of K and V tiles
  static constexpr int RAW = E4M3 ? 128 * D : 0, RS = D == 64 ? 4 : 3;      // ring of 8-bit tiles, rows D bytes apart, pieces permuted as the copy engine does
  static constexpr int LAG = 1;                                 // gathered tiles whose copies may be in flight when the next is begun
  static constexpr int NV = 8;                                  // ring of the keys' validity, by step
  static constexpr int Q_AT = 0, RING_AT = NT * Q_TILE, RAW_AT = RING_AT + NST * TILE, CTRL_AT = RAW_AT + RS * RAW;
  static constexpr int SMEM = CTRL_AT + 640;
  static_assert(BLOCKS * (SMEM + 1024) <= 228 * 1024, "blocks of an SM");
  static __device__ __forceinline__ uint32_t q_at(int row, int chunk) { return (uint32_t)((chunk >> 3) * Q_PART + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)); }
  static __device__ __forceinline__ uint32_t raw_at(int row, int chunk) {      // a 16-byte piece of an 8-bit row
    return D == 64 ? (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4)) : (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4));
  }
};
struct TcCtrl {
  u64 q_full, full[8], empty[8], s_full[2], s_free[2], pa_full[2], p_full[2], o_full[2];      // a: the first half
  u64 look[8];                                                  // bf16: a tile that the workers look through has landed
  u64 raw_full[4], raw_empty[4];
  uint32_t tmem, dead;
  int odd_lo, odd_hi;
  alignas(16) uint8_t valid[8][16];                             // by step, a bit for each key
};
static_assert(sizeof(TcCtrl) <= 640, "control area");

constexpr float BIG = 1073741824.f;                             // 2^30

__device__ __forceinline__ bool elect_one() {                  // one thread of a converged warp
  uint32_t e;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e != 0;
}
// D[tmem] (+)= A[tmem] * B[smem desc]
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, u64 desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
template <bool INC, int N> __device__ __forceinline__ void set_regs() {
  if constexpr (INC) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, int n) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n) : "memory"); }
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }      // the lowest n bits
__device__ __forceinline__ uint32_t tile_at(int row, int chunk) { return (uint32_t)((chunk >> 3) * 16384 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)); }

template <int D, bool E4M3, int NT>
__global__ void __launch_bounds__(Tc<D, E4M3, NT>::THREADS, Tc<D, E4M3, NT>::BLOCKS) many_rows_kernel(const __grid_constant__ AttnArgs P) {
  using F = Tc<D, E4M3, NT>;
  constexpr int WK = F::WORKERS;
  extern __shared__ __align__(1024) unsigned char smem[];       // the swizzle's atoms
  TcCtrl& ct = *reinterpret_cast<TcCtrl*>(smem + F::CTRL_AT);
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  after_the_kernel_before();
  // The last tiles, which have the most keys, start first: over all sequences and heads, or, where their keys and values together would not stay in L2, head by head
  const int split = (int)blockIdx.x % P.nsplit, rest = (int)blockIdx.x / P.nsplit, streams = P.n_kv_heads * P.b.n_seqs;
  const int turn = P.by_head ? rest % P.tiles : rest / streams, stream = P.by_head ? rest / P.tiles : rest % streams, kvh = stream % P.n_kv_heads;
  const int seq = P.ranked ? by_length(P.b, stream / P.n_kv_heads, reinterpret_cast<int*>(smem)) : stream / P.n_kv_heads;      // where Q will be
  const Chunk ch = chunk_of(P.b, seq);
  const int group = (int)P.group.d, cap = reach(P.b, ch.len);
  if (ch.len > cap && tid == 0) flag(P.b.status, ST_LENGTH);
  const int npair = (ch.n * group + NT * F::ROWS - 1) / (NT * F::ROWS);      // pairs of tiles, or tiles
  if (turn >= npair) return;
  if (tid == 0) {
    mbar_init(smem_u32(&ct.q_full), 4 * NT);
    for (int s = 0; s < F::NST; s++) { mbar_init(smem_u32(&ct.full[s]), F::WORKERS); mbar_init(smem_u32(&ct.empty[s]), NT); mbar_init(smem_u32(&ct.look[s]), 1); }
    for (int s = 0; s < 4; s++) { mbar_init(smem_u32(&ct.raw_full[s]), 1); mbar_init(smem_u32(&ct.raw_empty[s]), F::WORKERS); }
    for (int i = 0; i < NT; i++) {
      mbar_init(smem_u32(&ct.s_full[i]), 1); mbar_init(smem_u32(&ct.s_free[i]), 4);
      mbar_init(smem_u32(&ct.pa_full[i]), 4); mbar_init(smem_u32(&ct.p_full[i]), 4); mbar_init(smem_u32(&ct.o_full[i]), 1);
    }
    ct.odd_lo = 0x7fffffff; ct.odd_hi = -1; ct.dead = 0;
    mbar_fence_init();
  }
  if (warp == 4 * NT) tmem_alloc(smem_u32(&ct.tmem), F::TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ct.tmem;
  // Steps of 128 keys that the block walks for a pair of tiles, and those [a, b) that each tile takes part in
  struct Walk { int a[NT], b[NT], lo, hi, A, B, p_low, p_high; };
  auto walk = [&](int pair) {
    Walk k;
    k.lo = 0x7fffffff; k.hi = 0; k.p_low = k.p_high = 0;
#pragma unroll
    for (int i = 0; i < NT; i++) {
      const int r0 = (pair * NT + i) * F::ROWS;
      if (r0 >= ch.n * group) { k.a[i] = k.b[i] = 0; continue; }
      const int pmin = ch.p0 + (int)P.group.quot(r0), pmax = ch.p0 + min(ch.n - 1, (int)P.group.quot(r0 + F::ROWS - 1));
      const int h = min(cap, P.causal ? pmax + 1 : ch.len), l = first_seen(P, pmin);
      if (i == 0) k.p_low = pmin;
      k.p_high = pmax;
      k.a[i] = l / 128; k.b[i] = h > l ? (h + 127) / 128 : k.a[i];
      if (h > l) { k.lo = min(k.lo, l); k.hi = max(k.hi, h); }
    }
    if (k.lo > k.hi) k.lo = k.hi;
    const int first = k.lo / 128, nst = k.hi > k.lo ? (k.hi + 127) / 128 - first : 0;
    k.A = first + (int)((long long)nst * split / P.nsplit); k.B = first + (int)((long long)nst * (split + 1) / P.nsplit);
#pragma unroll
    for (int i = 0; i < NT; i++) { k.a[i] = max(k.a[i], k.A); k.b[i] = max(k.a[i], min(k.b[i], k.B)); }
    return k;
  };
  // a step that not every row of the block sees whole
  auto partial = [&](const Walk& k, int j) {
    return j * 128 < k.lo || j * 128 + 128 > k.hi || (P.causal && j * 128 + 127 > k.p_low) || j * 128 < first_seen(P, k.p_high);
  };
  // the end of a pair for all warps: tiles, control words and tensor memory are free for the next; false: a wait ran out somewhere
  auto next = [&](bool ok) {
    if (!ok) { atomicExch(&ct.dead, 1u); flag(P.b.status, ST_TIMEOUT); }
    __syncthreads();
    const bool go = ct.dead == 0;
    if (tid == 0) { ct.odd_lo = 0x7fffffff; ct.odd_hi = -1; }
    tc_fence_after();
    __syncthreads();
    return go;
  };
  bool ok = true;

  if (warp < 4 * NT) {
    // ------------------------------------------------------------------------------------------ softmax: a thread a row
    set_regs<true, F::SOFT_REGS>();
    const int tile = warp >> 2, e = warp & 3, r = e * 32 + lane;
    uint32_t done = 0;                                           // steps of this tile so far: phases of its barriers
    for (int pair = npair - 1 - turn; pair >= 0; pair -= P.tiles) {
      const Walk k = walk(pair);
      const int rr = (pair * NT + tile) * F::ROWS + r, t = (int)P.group.quot(rr);
      const bool on = r < F::ROWS && t < ch.n;
      const int pos = ch.p0 + (on ? t : ch.n - 1), head = kvh * group + rr - t * group;
      unsigned char* qt = smem + F::Q_AT + tile * F::Q_TILE;
      constexpr int CQ = D / 8;                                  // 16-byte pieces of a row
      const bool idle = e * 32 >= F::ROWS || (pair * NT + tile) * F::ROWS + e * 32 >= ch.n * group;      // none of the warp's rows is there: whatever is computed for them is not looked at
      if (!idle) {                                               // the warp's 32 rows of Q, whole rows side by side
        const long long at = on ? (long long)(ch.s + t) * P.q_row + (long long)head * P.q_head : -1;
#pragma unroll 4
        for (int q = 0; q < CQ; q++) {
          const long long o = __shfl_sync(0xffffffffu, at, (q * 32 + lane) / CQ);
          cp16(smem_u32(qt) + F::q_at(e * 32 + (q * 32 + lane) / CQ, lane % CQ), P.q + (o >= 0 ? o : 0) + lane % CQ * 8, o >= 0);
        }
        cp_commit();
        cp_wait<0>();
        fence_async_shared();
      }
      attn_tc::warp_arrive(smem_u32(&ct.q_full));
      const uint32_t tl = tmem + ((uint32_t)(e * 32) << 16), ts = tl + tile * 128, to = tl + F::O_AT + tile * D;
      float m = -INFINITY, l = 0.f, sc = P.scale_log2;
      const int n = k.b[tile] - k.a[tile];
      for (int c = 0; c < n; c++) {
        const int j = k.a[tile] + c, k0 = j * 128;
        if (idle) {
          ok = wait_for(smem_u32(&ct.s_full[tile]), (done + c) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          attn_tc::warp_arrive(smem_u32(&ct.s_free[tile]));
          attn_tc::warp_arrive(smem_u32(&ct.pa_full[tile]));
          attn_tc::warp_arrive(smem_u32(&ct.p_full[tile]));
          continue;
        }
        uint32_t s[4][32];
        ok = wait_for(smem_u32(&ct.s_full[tile]), (done + c) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        attn_tc::tmem_ld32_nw(ts, s[0]);
        attn_tc::tmem_ld32_nw(ts + 32, s[1]);
        attn_tc::tmem_ld32_nw(ts + 64, s[2]);
        attn_tc::tmem_ld32_nw(ts + 96, s[3]);
        attn_tc::tmem_ld_wait();
        tc_fence_before();
        attn_tc::warp_arrive(smem_u32(&ct.s_free[tile]));        // the first half of the next scores may overwrite these
        const uint4 vw = *reinterpret_cast<const uint4*>(ct.valid[j % F::NV]);
        if (partial(k, j) || (vw.x & vw.y & vw.z & vw.w) != 0xffffffffu) {
          const int x1 = P.causal ? pos - k0 : 127, x0 = first_seen(P, pos) - k0;       // of the step's keys the row sees x0 .. x1
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const uint32_t w = (q == 0 ? vw.x : q == 1 ? vw.y : q == 2 ? vw.z : vw.w) & below(x1 + 1 - q * 32) & ~below(x0 - q * 32);
#pragma unroll
            for (int x = 0; x < 32; x++) s[q][x] = w & (1u << x) ? s[q][x] : 0xff800000u;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < 32; x += 2)
#pragma unroll
          for (int q = 0; q < 4; q++) mx[q] = attn_tc::max3(mx[q], __uint_as_float(s[q][x]), __uint_as_float(s[q][x + 1]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), m_true = fmaxf(m, top * sc);
        // The multiply-add below forms products exactly, the reference is a rounded one: the largest score's exponent is up to half a step of the reference off 0, which from 2^31 on is more
        // than sums have room for. Beyond 2^30, where two scores that are not alike lie 2^6 or more apart, the factor is its power of two instead, whose products are exact.
        auto factor = [&](float x) { return fabsf(x * P.scale_log2) > BIG && x != -INFINITY ? __uint_as_float(__float_as_uint(P.scale_log2) & 0xff800000u) : P.scale_log2; };
        if (c == 0) { sc = factor(top); m = top * sc; }
        else {
          const bool grow = m_true > m + RESCALE_LOG2;
          if (__any_sync(0xffffffffu, grow)) {
            float alpha = grow ? ex2_approx(m - m_true) : 1.f;
            if (grow) {
              const float f = factor(top);
              if (f != sc) alpha = 0.f;                          // the old reference is 2^5 or more below the new one
              sc = f; m = top * sc; l *= alpha;
            }
#pragma unroll 1
            for (int q = 0; q < D / 16; q++) {
              uint32_t o[16];
              attn_tc::tmem_ld16(to + q * 16, o);
#pragma unroll
              for (int x = 0; x < 16; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
              attn_tc::tmem_st16(to + q * 16, o);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;              // no key seen yet: 2^(-inf - 0) = 0
        const u64 sc2 = attn_tc::f2(sc, sc), nm2 = attn_tc::f2(-ref, -ref);
        u64 sum[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 4; q++) {
          uint32_t pk[16];
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            const float2 v = attn_tc::unf2(attn_tc::fma2(attn_tc::f2(__uint_as_float(s[q][x]), __uint_as_float(s[q][x + 1])), sc2, nm2));
            const float p0 = ex2_approx(v.x), p1 = ex2_approx(v.y);
            sum[(x >> 1) & 1] = attn_tc::add2(sum[(x >> 1) & 1], attn_tc::f2(p0, p1));
            pk[x >> 1] = pack2f(p0, p1);                         // rounded to bf16 for the product; the sum is taken before
          }
          attn_tc::tmem_st16(ts + 64 + q * 16, pk);
          if (q == 1) {
            attn_tc::tmem_st_wait();
            tc_fence_before();
            attn_tc::warp_arrive(smem_u32(&ct.pa_full[tile]));
          }
        }
        attn_tc::tmem_st_wait();
        tc_fence_before();
        attn_tc::warp_arrive(smem_u32(&ct.p_full[tile]));
        const float2 s0 = attn_tc::unf2(attn_tc::add2(sum[0], sum[1]));
        l += s0.x + s0.y;
      }
      if (ok && n > 0) {
        ok = wait_for(smem_u32(&ct.o_full[tile]), (done + n - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (sc != P.scale_log2) m = m / sc * P.scale_log2;
      if (ok && !idle) {                                         // the row's result, or its part for combine_kernel
        const int olo = *reinterpret_cast<volatile int*>(&ct.odd_lo), ohi = *reinterpret_cast<volatile int*>(&ct.odd_hi);
        const long long g = (long long)(ch.s + t) * P.n_heads + head;
        const float inv = P.nsplit > 1 || !on ? 1.f : over(P, l, seq, pos);
#pragma unroll 1
        for (int q = 0; q < D / 32; q++) {
          uint32_t o[32];
          if (n > 0) tmem_ld32(to + q * 32, o);
          else {
#pragma unroll
            for (int x = 0; x < 32; x++) o[x] = 0;
          }
          if (ohi >= olo) {                                      // rare: what the loaders left out
            for (int key = olo; key <= ohi; key++) {
              int page, at;
              if ((P.causal && key > pos) || key < first_seen(P, pos) || key / 128 < k.a[tile] || key / 128 >= k.b[tile] || !locate(P.b, seq, key, page, at)) continue;
              const char* row = P.c.v + (long long)kvh * P.c.head_b + (long long)page * P.c.page_b + (long long)at * P.c.row_b;
              const int sc = E4M3 ? P.c.vs[(long long)page * P.c.s_page + (long long)kvh * P.c.s_head + (long long)at * P.c.s_row] : 0;
#pragma unroll
              for (int x = 0; x < 32; x++) {
                const float v = held<E4M3>(row, q * 32 + x, sc);
                if (!isfinite(v)) o[x] = __float_as_uint(__uint_as_float(o[x]) + v);
              }
            }
            __syncwarp();                                        // tensor memory is read by whole warps
          }
          if (P.nsplit == 1) {                                   // through the tile of Q, which is not needed any more, so that rows leave whole
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
              float f[8];
#pragma unroll
              for (int y = 0; y < 8; y++) f[y] = __uint_as_float(o[x + y]) * inv;
              *reinterpret_cast<uint4*>(qt + F::q_at(r, (q * 32 + x) / 8)) = pack8(f);
            }
          } else {                                               // 128 bytes of each of the warp's rows, the same way
            unsigned char* mine = qt + e * 4096;
#pragma unroll
            for (int x = 0; x < 8; x++) *reinterpret_cast<uint4*>(mine + lane * 128 + ((x ^ (lane & 7)) << 4)) = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 8; x++) {
              const int row = x * 4 + (lane >> 3);
              const long long d = __shfl_sync(0xffffffffu, on ? g : -1ll, row);
              if (d >= 0) *reinterpret_cast<uint4*>(P.part + (d * P.nsplit + split) * D + q * 32 + (lane & 7) * 4) = *reinterpret_cast<const uint4*>(mine + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
            }
            __syncwarp();
          }
        }
        if (P.nsplit == 1) {
          __syncwarp();
          const long long at = on ? (long long)(ch.s + t) * P.o_row + (long long)head * P.o_head : -1;
#pragma unroll 4
          for (int q = 0; q < CQ; q++) {
            const long long d = __shfl_sync(0xffffffffu, at, (q * 32 + lane) / CQ);
            if (d >= 0) *reinterpret_cast<uint4*>(P.out + d + lane % CQ * 8) = *reinterpret_cast<const uint4*>(qt + F::q_at(e * 32 + (q * 32 + lane) / CQ, lane % CQ));
          }
        }
        if (on && P.nsplit > 1) reinterpret_cast<float2*>(P.part + (long long)P.b.n_rows * P.n_heads * P.nsplit * D)[g * P.nsplit + split] = make_float2(m, l);
        else if (on && P.lse) P.lse[g] = l == 0.f ? -INFINITY : m * LN2 + logf(l);
      }
      tc_fence_before();
      done += (uint32_t)n;
      if (!next(ok)) break;
    }
  } else if (warp < 5 * NT) {
    // ------------------------------------------------------------------------------------------ products
    set_regs<false, F::REST_REGS>();
    const int tile = warp - 4 * NT;
    uint32_t uses = 0, done = 0, round = 0;                      // items through the ring, steps of the tile
    // The whole warp walks, so that descriptors and addresses stay uniform, and one elected thread issues. What the loaders wrote is ordered before
    // the products' reads by a fence here: in the loaders it would wait for every copy they have in flight.
    const bool leader = elect_one();
    for (int pair = npair - 1 - turn; pair >= 0; pair -= P.tiles) {
      const Walk k = walk(pair);
      const int ka = k.a[tile], kb = k.b[tile];
      const uint32_t ts = tmem + tile * 128, to = tmem + F::O_AT + tile * D;
      const u64 dq = umma_smem_desc(base + F::Q_AT + tile * F::Q_TILE, 16, 1024);
      const uint32_t I_S = umma_idesc(false, false, 128, 64) | (uint32_t)P.flip << 13;      // negates Q where scores are scaled by a negative number
      constexpr uint32_t I_O = umma_idesc(false, true, 128, D);
      uint32_t c = 0;
      auto slot_of = [&](int item) { return (uses + (uint32_t)item) % F::NST; };
      auto filled = [&](int item) { return wait_for(smem_u32(&ct.full[slot_of(item)]), ((uses + (uint32_t)item) / F::NST) & 1); };
      auto scores = [&](int j, int half) {                       // S = Q K_j^T for 64 keys; one thread's products run in their order
        const uint32_t slot = slot_of(2 * (j - k.A));
        const u64 dk = umma_smem_desc(base + F::RING_AT + slot * F::TILE + half * 8192, 16, 1024);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++)
            umma_bf16(ts + half * 64, dq + ((kk >> 2) * F::Q_PART + (kk & 3) * 32) / 16, dk + ((kk >> 2) * 16384 + (kk & 3) * 32) / 16, I_S, kk > 0 ? 1u : 0u);
          if (half) { umma_commit(smem_u32(&ct.s_full[tile])); umma_commit(smem_u32(&ct.empty[slot])); }
        }
      };
      auto pass = [&](int item) {                                // a tile that this issuer has no use for
        if (!filled(item)) return false;
        if (leader) mbar_arrive(smem_u32(&ct.empty[slot_of(item)]));
        return true;
      };
      ok = wait_for(smem_u32(&ct.q_full), round & 1);
      for (int item = 0; item < 2 * ((kb > ka ? ka : k.B) - k.A) && ok; item++) ok = pass(item);
      if (ka < kb && ok) {
        ok = filled(2 * (ka - k.A));
        fence_async_shared();                                    // what the workers wrote, before it is read by the products
        if (ok) { scores(ka, 0); scores(ka, 1); }
      }
      for (int j = ka; j < kb && ok; j++, c++) {
        const int item = 2 * (j - k.A) + 1;
        ok = filled(item) && (j + 1 == kb || filled(item + 1));
        if (!ok) break;
        fence_async_shared();
        if (j + 1 < kb) {
          ok = wait_for(smem_u32(&ct.s_free[tile]), (done + c) & 1);
          if (!ok) break;
          tc_fence_after();
          scores(j + 1, 0);
        }
        const uint32_t slot = slot_of(item);
        const u64 dv = umma_smem_desc(base + F::RING_AT + slot * F::TILE, 16384, 1024);
#pragma unroll
        for (int half = 0; half < 2; half++) {                   // O += P V_j
          ok = ok && wait_for(smem_u32(half ? &ct.p_full[tile] : &ct.pa_full[tile]), (done + c) & 1);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int kk = half * 4; kk < half * 4 + 4; kk++) umma_bf16_ts(to, ts + 64 + kk * 8, dv + kk * 2048 / 16, I_O, (c > 0 || kk > 0) ? 1u : 0u);
          }
        }
        if (!ok) break;
        if (leader) {
          umma_commit(smem_u32(&ct.o_full[tile]));
          umma_commit(smem_u32(&ct.empty[slot]));
        }
        if (j + 1 < kb) scores(j + 1, 1);
      }
      if (kb > ka) for (int item = 2 * (kb - k.A); item < 2 * (k.B - k.A) && ok; item++) ok = pass(item);
      uses += 2u * (uint32_t)(k.B - k.A); done += (uint32_t)(kb - ka); round++;
      if (!next(ok)) break;
    }
  } else if (warp == 5 * NT) {
    // ------------------------------------------------------------------------------------------ copies
    set_regs<false, F::REST_REGS>();
    const int run = P.run ? P.run : 8, nrun = 128 / run;         // a lane for each run of a step's keys
    uint32_t uses = 0;
    for (int pair = npair - 1 - turn; pair >= 0; pair -= P.tiles) {
      const Walk k = walk(pair);
      if (P.run) {
        auto reaches = [&](int j) { const int key = j * 128 + lane * run; return lane < nrun && j < k.B && key + run > k.lo && key < k.hi; };
        auto page_of = [&](int j) { return reaches(j) ? __ldg(P.b.pages + (long long)seq * P.b.pages_stride + P.b.page.quot((unsigned)(j * 128 + lane * run))) : -1; };      // below cap
        int page = page_of(k.A);
        for (int j = k.A; j < k.B && ok; j++) {
          const int pg = page, key = j * 128 + lane * run, at = key - (int)(P.b.page.quot((unsigned)key) * P.b.page.d);
          page = page_of(j + 1);
          const bool there = (unsigned)pg < (unsigned)P.b.n_pages, bad = reaches(j) && !there;
          if (bad) flag(P.b.status, ST_PAGE);
          const bool any_bad = __any_sync(0xffffffffu, bad);
          const uint32_t there_runs = __ballot_sync(0xffffffffu, there), bytes = __popc(there_runs) * (uint32_t)(run * D * (E4M3 ? 1 : 2));
#pragma unroll
          for (int half = 0; half < 2; half++) {
            const uint32_t n = uses + 2 * (uint32_t)(j - k.A) + half, slot = n % F::NST, rs = n % F::RS;
            if constexpr (E4M3) ok = wait_for(smem_u32(&ct.raw_empty[rs]), ((n / F::RS) & 1) ^ 1);
            else ok = wait_for(smem_u32(&ct.empty[slot]), ((n / F::NST) & 1) ^ 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (half == 0) {                                     // which keys are there, eight a lane
              const int key8 = j * 128 + lane * 8;
              const bool t8 = (there_runs >> (lane * 8 / run & 31)) & 1;
              if (lane < 16) ct.valid[j % F::NV][lane] = t8 ? (uint8_t)(below(k.hi - key8) & ~below(k.lo - key8)) : 0;
            }
            const CUtensorMap* map = half ? &P.vm : &P.km;
            if constexpr (E4M3) {
              if (lane == 0) mbar_expect_tx(smem_u32(&ct.raw_full[rs]), bytes);
              __syncwarp();
              if (there) tma_load_4d(base + F::RAW_AT + rs * F::RAW + lane * run * D, map, smem_u32(&ct.raw_full[rs]), 0, at, kvh, pg);
            } else {
              unsigned char* dst = smem + F::RING_AT + slot * F::TILE;
              if (half && any_bad) {                             // values of rows that are not there: zeros
                if (bad)
                  for (int x = 0; x < run * 8; x++)
                    for (int h = 0; h < D / 64; h++) *reinterpret_cast<uint4*>(dst + h * 16384 + lane * run * 128 + x * 16) = make_uint4(0, 0, 0, 0);
                fence_async_shared();
                __syncwarp();
              }
              const bool look = half && partial(k, j);
              const uint32_t bar = smem_u32(look ? &ct.look[slot] : &ct.full[slot]);
              if (lane == 0) {
                if (!look) mbar_arrive_n(bar, F::WORKERS - 1);
                mbar_expect_tx(bar, bytes);
              }
              __syncwarp();
              if (there) {
#pragma unroll
                for (int h = 0; h < D / 64; h++) tma_load_4d(base + F::RING_AT + slot * F::TILE + h * 16384 + lane * run * 128, map, bar, h * 64, at, kvh, pg);
              }
            }
          }
        }
      }
      uses += 2u * (uint32_t)(k.B - k.A);
      if (!next(ok)) break;
    }
  } else if (warp > 5 * NT + WK) {
    set_regs<false, F::REST_REGS>();
    for (int pair = npair - 1 - turn; pair >= 0; pair -= P.tiles) if (!next(true)) break;
  } else {
    // ------------------------------------------------------------------------------------------ workers
    set_regs<false, F::REST_REGS>();
    const int w = warp - 5 * NT - 1;
    constexpr int CH = E4M3 ? D / 16 : D / 8, IT = 8 * CH / 32 > 0 ? 8 * CH / 32 : 1;      // 16-byte pieces of a held row; of 8 rows, for each lane
    constexpr int LAG = F::LAG;
    const char* kbase = P.c.k + (long long)kvh * P.c.head_b;
    const char* vbase = P.c.v + (long long)kvh * P.c.head_b;
    uint32_t uses = 0, looks = 0;                                // looks: a bit for each slot, the phase of its barrier
    // A span's 128 keys are 16 units of 8 rows, dealt out to the workers through all items: unit e of all is e % 16 of item e / 16 and the work of worker e % WORKERS. A
    // lane places one row, up to four units of an item at once: its page is asked for two items ahead, its scale one.
    constexpr int UNITS = (16 + WK - 1) / WK, GROUPS = (UNITS + 3) / 4;
    struct Row { int page, at; };
    for (int pair = npair - 1 - turn; pair >= 0; pair -= P.tiles) {
      const Walk k = walk(pair);
      const int total = 2 * (k.B - k.A);
      auto unit0 = [&](int item) { return (w + WK - item * 16 % WK) % WK; };               // the first unit of this worker
      auto row_of = [&](int item, int gr) {                                                // this lane's row of its unit number gr * 4 + lane / 8; its page is not looked at yet
        const int u = unit0(item) + (gr * 4 + (lane >> 3)) * WK, key = (k.A + (item >> 1)) * 128 + u * 8 + (lane & 7);
        Row x = {-1, 0};
        if (item < total && u < 16 && key >= k.lo && key < k.hi) {                         // below cap: within the table
          const unsigned idx = P.b.page.quot((unsigned)key);
          x.at = key - (int)(idx * P.b.page.d);
          x.page = __ldg(P.b.pages + (long long)seq * P.b.pages_stride + idx);
          x.at |= 1 << 31;                                                                 // there should be one
        }
        return x;
      };
      auto known = [&](Row x) {                                                            // and now it is
        const bool want = x.at < 0;
        x.at &= 0x7fffffff;
        if (want && (unsigned)x.page >= (unsigned)P.b.n_pages) { flag(P.b.status, ST_PAGE); x.page = -1; }
        if (!want) x.page = -1;
        return x;
      };
      auto offset = [&](const Row& x) { return x.page >= 0 ? (long long)x.page * P.c.page_b + (long long)x.at * P.c.row_b : -1ll; };
      // A row's scale byte as it comes from memory: anything done with it here would wait for it
      auto scale = [&](const Row& x, int item) {
        unsigned char s = 0;
        if (x.page >= 0) s = __ldg((item & 1 ? P.c.vs : P.c.ks) + (long long)x.page * P.c.s_page + (long long)kvh * P.c.s_head + (long long)x.at * P.c.s_row);
        return s;
      };
      auto odd_at = [&](int key) { atomicMin(&ct.odd_lo, key); atomicMax(&ct.odd_hi, min(k.hi - 1, key)); };
      auto tile_free = [&](int item) {
        const uint32_t n = uses + (uint32_t)item;
        ok = wait_for(smem_u32(&ct.empty[n % F::NST]), ((n / F::NST) & 1) ^ 1);
        ok = __all_sync(0xffffffffu, ok);
        return ok;
      };
      auto done_with = [&](int item) { attn_tc::warp_arrive(smem_u32(&ct.full[(uses + (uint32_t)item) % F::NST])); };
      if constexpr (E4M3) {
        // 8-bit rows, from their ring; where the copy engine does not bring them, by this warp's own copies, RS - 1 items ahead
        auto gather = [&](int item) {
          if (item < total) {
            const uint32_t n = uses + (uint32_t)item, rs = n % F::RS;
            ok = ok && wait_for(smem_u32(&ct.raw_empty[rs]), ((n / F::RS) & 1) ^ 1);       // the rows that this warp writes there are others than it read
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
#pragma unroll 1
            for (int gr = 0; gr < GROUPS; gr++) {
              const long long off = offset(known(row_of(item, gr)));
              const uint32_t there = __ballot_sync(0xffffffffu, off >= 0);
#pragma unroll 1
              for (int y = 0; y < 4; y++) {
                const int u = unit0(item) + (gr * 4 + y) * WK;
                if (GROUPS * 4 * WK != 16 && u >= 16) break;
                if (!(item & 1) && lane == 0) ct.valid[(k.A + (item >> 1)) % F::NV][u] = (uint8_t)(there >> y * 8);
                long long o[IT];
#pragma unroll
                for (int i = 0; i < IT; i++) o[i] = from_lane(off, y * 8 + ((i * 32 + lane) / CH & 7), P.wide);
#pragma unroll
                for (int i = 0; i < IT; i++)
                  cp16(base + F::RAW_AT + rs * F::RAW + F::raw_at(u * 8 + (i * 32 + lane) / CH, lane % CH), (item & 1 ? vbase : kbase) + (o[i] >= 0 ? o[i] : 0) + lane % CH * 16, o[i] >= 0);
              }
            }
          }
          cp_commit();
        };
        if (!P.run) for (int i = 0; i < F::RS - 1; i++) gather(i);
        Row ahead[GROUPS];
        unsigned char next_f[GROUPS];
        bool next_there[GROUPS];
#pragma unroll
        for (int gr = 0; gr < GROUPS; gr++) {
          const Row x = known(row_of(0, gr));
          next_f[gr] = scale(x, 0); next_there[gr] = x.page >= 0; ahead[gr] = row_of(1, gr);
        }
        for (int item = 0; item < total && ok; item++) {
          const uint32_t n = uses + (uint32_t)item, rs = n % F::RS;
          const int j = k.A + (item >> 1);
          const bool check = (item & 1) && partial(k, j);
          if (P.run) ok = wait_for(smem_u32(&ct.raw_full[rs]), (n / F::RS) & 1);
          else { gather(item + F::RS - 1); cp_wait<F::RS - 1>(); __syncwarp(); }
          if (!__all_sync(0xffffffffu, ok) || !tile_free(item)) { ok = false; break; }
          uint32_t f[GROUPS];                                    // 2^120 times the scale, as bf16; 0: rows that are not there become zeros
#pragma unroll
          for (int gr = 0; gr < GROUPS; gr++) {
            f[gr] = next_there[gr] ? scale_bits((int)next_f[gr]) : 0u;
            const Row x = known(ahead[gr]);
            next_f[gr] = scale(x, item + 1); next_there[gr] = x.page >= 0;
            ahead[gr] = row_of(item + 2, gr);
          }
          const unsigned char* src = smem + F::RAW_AT + rs * F::RAW;
          unsigned char* dst = smem + F::RING_AT + n % F::NST * F::TILE;
#pragma unroll
          for (int gr = 0; gr < GROUPS; gr++) {
            uint32_t mine = f[gr];
            if (check && mine == 0x7fc0u) { odd_at(j * 128 + (unit0(item) + (gr * 4 + (lane >> 3)) * WK) * 8 + (lane & 7)); mine = 0; }
            mine |= mine << 16;
#pragma unroll
            for (int y = 0; y < 4; y++) {
              const int u = unit0(item) + (gr * 4 + y) * WK;
              if (GROUPS * 4 * WK != 16 && u >= 16) break;
#pragma unroll
              for (int i = 0; i < IT; i++) {
                // rows of 8 pieces in pairs, half of each to eight lanes, which then write to all the banks: two pieces of a tile's row lie side by side
                const int row = CH == 8 ? i * 4 + ((lane >> 3) ^ (lane >> 2 & 1)) : (i * 32 + lane) / CH, q = lane % CH, r = u * 8 + row;
                const uint32_t fr = __shfl_sync(0xffffffffu, mine, y * 8 + row);
                const uint4 v = *reinterpret_cast<const uint4*>(src + F::raw_at(r, q));
                *reinterpret_cast<uint4*>(dst + tile_at(r, 2 * q)) = make_uint4(widen_lo(v.x, fr), widen_hi(v.x, fr), widen_lo(v.y, fr), widen_hi(v.y, fr));
                *reinterpret_cast<uint4*>(dst + tile_at(r, 2 * q + 1)) = make_uint4(widen_lo(v.z, fr), widen_hi(v.z, fr), widen_lo(v.w, fr), widen_hi(v.w, fr));
              }
            }
          }
          done_with(item);
          attn_tc::warp_arrive(smem_u32(&ct.raw_empty[rs]));
        }
      } else if (P.run) {
        // look through the values of steps that not every row sees whole
        for (int j = k.A; j < k.B && ok; j++) {
          if (!partial(k, j)) continue;
          const int item = 2 * (j - k.A) + 1;
          const uint32_t slot = (uses + (uint32_t)item) % F::NST;
          ok = wait_for(smem_u32(&ct.look[slot]), looks >> slot & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          looks ^= 1u << slot;
          unsigned char* tile = smem + F::RING_AT + slot * F::TILE;
#pragma unroll 4
          for (int c = w * 32 + lane; c < F::TILE / 16; c += F::WORKERS * 32) {
            const uint4 u = *reinterpret_cast<const uint4*>(tile + c * 16);
            if (odd_bits(u.x) || odd_bits(u.y) || odd_bits(u.z) || odd_bits(u.w)) {
              *reinterpret_cast<uint4*>(tile + c * 16) = make_uint4(without_odd(u.x), without_odd(u.y), without_odd(u.z), without_odd(u.w));
              const int row = (c * 16 & 16383) / 128;            // what lies behind the context in its last page counts nowhere
              if (ct.valid[j % F::NV][row >> 3] >> (row & 7) & 1) odd_at(j * 128 + row);
            }
          }
          done_with(item);
        }
      } else {
        // gather
        Row now[GROUPS];
#pragma unroll
        for (int gr = 0; gr < GROUPS; gr++) now[gr] = row_of(0, gr);
        for (int item = 0; item < total + LAG && ok; item++) {
          if (item < total) {
            if (!tile_free(item)) break;
            const int j = k.A + (item >> 1);
            const char* src = item & 1 ? vbase : kbase;
            const uint32_t slot = (uses + (uint32_t)item) % F::NST;
            unsigned char* dst = smem + F::RING_AT + slot * F::TILE;
            const bool check = (item & 1) && partial(k, j);
#pragma unroll
            for (int gr = 0; gr < GROUPS; gr++) {
              const long long off = offset(known(now[gr]));
              now[gr] = row_of(item + 1, gr);
              const uint32_t there = __ballot_sync(0xffffffffu, off >= 0);
#pragma unroll 1
              for (int y = 0; y < 4; y++) {
                const int u = unit0(item) + (gr * 4 + y) * WK;
                if (GROUPS * 4 * WK != 16 && u >= 16) break;
                if (!(item & 1) && lane == 0) ct.valid[j % F::NV][u] = (uint8_t)(there >> y * 8);
                long long o[IT];                                 // all the exchanges before the first copy: in turns each copy would wait for its own
#pragma unroll
                for (int i = 0; i < IT; i++) o[i] = from_lane(off, y * 8 + (i * 32 + lane) / CH, P.wide);
#pragma unroll
                for (int i = 0; i < IT; i++) {
                  const int row = u * 8 + (i * 32 + lane) / CH, q = lane % CH;
                  if (!check) cp16(smem_u32(dst) + tile_at(row, q), src + (o[i] >= 0 ? o[i] : 0) + q * 16, o[i] >= 0);
                  else {
                    uint4 v = o[i] >= 0 ? *reinterpret_cast<const uint4*>(src + o[i] + q * 16) : make_uint4(0, 0, 0, 0);
                    if (odd_bits(v.x) || odd_bits(v.y) || odd_bits(v.z) || odd_bits(v.w)) {
                      odd_at(j * 128 + row);
                      v = make_uint4(without_odd(v.x), without_odd(v.y), without_odd(v.z), without_odd(v.w));
                    }
                    *reinterpret_cast<uint4*>(dst + tile_at(row, q)) = v;
                  }
                }
              }
            }
          }
          cp_commit();
          cp_wait<LAG>();
          if (item >= LAG) done_with(item - LAG);
        }
      }
      cp_wait<0>();
      uses += (uint32_t)total;
      if (!next(ok)) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4 * NT) tmem_dealloc(tmem, F::TMEM);
}

}  // namespace paged
}  // namespace ofa
