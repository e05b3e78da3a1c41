// Attention of many rows over a paged cache on the 5th-generation tensor cores: chunks of new tokens, where the products count.
//
// The rows of a key/value head (new tokens x the query heads that share it) are taken 256 at a time by a block of 16 warps, two tiles of 128 rows that walk the
// same keys 128 at a time, half a step apart: while the softmax warps of one tile work, the tensor pipe works for the other.
//   warps 0-3, 4-7   softmax of tile 0 and 1, a thread per row (= tensor-memory lane): reads its 128 scores, keeps maximum and sum, writes the probabilities
//                    back over them as bf16, the A operand of the second product
//   warps 8, 9       one thread each issues a tile's products: S = Q K_j^T, then O += P V_j. Two threads because one issues a tcgen05.mma only every
//                    ~96 clocks, and a 128 x 128 x 16 product takes 64
//   warps 10-15      fetch keys and values into a ring of tiles in the layout the products read (128-byte swizzle)
// Tensor memory, 512 columns: S 0 / 128 (P in their last 64), O 256 / 256 + D. Rows of pages are gathered by cp.async, 16 bytes at a time, so pages
// may have any size and end inside a tile; 8-bit rows become bf16 in the loaders' registers, once for the 256 rows.
//
// A row's probabilities are taken against a reference that is raised only when the true maximum has passed it by 2^8 (they stay below 256: exact enough in fp32 sums and
// bf16), and only then is the row of O multiplied in tensor memory. Before S of the next step is issued the issuer has seen the product before it complete, so a softmax thread
// that has its scores may also rewrite its row of O.
//
// Keys that some rows of the block see and others do not (the diagonal, the window's edge, the end of the context) come in tiles whose loaders look at
// every value: infinities and NaN are left out and added at the end to the rows that see them.
#pragma once
#include "attn_tc.cuh"
#include "paged_attn.cuh"

namespace ofa {
namespace paged {

enum { ST_TIMEOUT = 8 };

template <int D> struct Tc {
  static constexpr int TILE = 128 * D * 2;                      // a tile of rows: D / 64 parts of 128 rows x 128 bytes
  static constexpr int NST = D == 128 ? 4 : 8;                  // ring of K and V tiles
  static constexpr int LAG = D == 128 ? 2 : 4;                  // tiles whose copies may be in flight when the next is begun
  static constexpr int NV = 8;                                  // ring of the keys' validity, by step
  static constexpr int Q_AT = 0, RING_AT = 2 * TILE, CTRL_AT = RING_AT + NST * TILE;
  static constexpr int SMEM = CTRL_AT + 512 + 1024;             // 1,024 for the alignment of the swizzle's atoms
  static constexpr int LOADERS = 6;
};
struct TcCtrl {
  u64 q_full, full[8], empty[8], s_full[2], p_full[2], o_full[2];
  uint32_t tmem, dead;
  int odd_lo, odd_hi;
  alignas(16) uint16_t valid[8][8];
};
static_assert(sizeof(TcCtrl) <= 512, "control area");

// A bounded wait without a call: a function with an ABI of its own does not go with setmaxnreg. A try sleeps for about 300 clocks, the limit is a second or a few.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 10000000; i++) if (mbar_try(bar, parity)) return true;
  return false;
}
template <bool INC, int N> __device__ __forceinline__ void set_regs() {
  if constexpr (INC) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ uint32_t tile_at(int row, int chunk) { return (uint32_t)((chunk >> 3) * 16384 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)); }

template <int D, bool E4M3>
__global__ void __launch_bounds__(512, 1) many_rows_kernel(const __grid_constant__ AttnArgs P) {
  using F = Tc<D>;
  extern __shared__ __align__(16) unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  TcCtrl& ct = *reinterpret_cast<TcCtrl*>(smem + F::CTRL_AT);
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the last pairs of tiles of a sequence have the most keys: they start first
  const int split = (int)blockIdx.x % P.nsplit, seq = (int)blockIdx.x / P.nsplit % P.b.n_seqs, kvh = blockIdx.y;
  const int turn = (int)blockIdx.x / P.nsplit / P.b.n_seqs;
  const Chunk ch = chunk_of(P.b, seq);
  const int group = (int)P.group.d, cap = (int)min((long long)P.b.max_pages * P.b.page.d, (long long)ch.len);
  if (ch.len > cap && tid == 0) flag(P.b.status, ST_LENGTH);
  const int npair = (ch.n * group + 255) / 256;
  if (turn >= npair) return;
  if (tid == 0) {
    mbar_init(smem_u32(&ct.q_full), 8);
    for (int s = 0; s < F::NST; s++) { mbar_init(smem_u32(&ct.full[s]), F::LOADERS); mbar_init(smem_u32(&ct.empty[s]), 2); }
    for (int i = 0; i < 2; i++) { mbar_init(smem_u32(&ct.s_full[i]), 1); mbar_init(smem_u32(&ct.p_full[i]), 4); mbar_init(smem_u32(&ct.o_full[i]), 1); }
    ct.odd_lo = 0x7fffffff; ct.odd_hi = -1; ct.dead = 0;
    mbar_fence_init();
  }
  if (warp == 8) tmem_alloc(smem_u32(&ct.tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ct.tmem;
  // Steps of 128 keys that the block walks for a pair of tiles, and those [a, b) that each tile takes part in
  struct Walk { int a[2], b[2], lo, hi, A, B, p_low, p_high; };
  auto walk = [&](int pair) {
    Walk k;
    k.lo = 0x7fffffff; k.hi = 0; k.p_low = k.p_high = 0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int r0 = (pair * 2 + i) * 128;
      if (r0 >= ch.n * group) { k.a[i] = k.b[i] = 0; continue; }
      const int pmin = ch.p0 + (int)P.group.quot(r0), pmax = ch.p0 + min(ch.n - 1, (int)P.group.quot(r0 + 127));
      const int h = min(cap, P.causal ? pmax + 1 : ch.len), l = P.window ? max(0, pmin - P.window + 1) : 0;
      if (i == 0) k.p_low = pmin;
      k.p_high = pmax;
      k.a[i] = l / 128; k.b[i] = h > l ? (h + 127) / 128 : k.a[i];
      if (h > l) { k.lo = min(k.lo, l); k.hi = max(k.hi, h); }
    }
    if (k.lo > k.hi) k.lo = k.hi;
    const int first = k.lo / 128, nst = k.hi > k.lo ? (k.hi + 127) / 128 - first : 0;
    k.A = first + (int)((long long)nst * split / P.nsplit); k.B = first + (int)((long long)nst * (split + 1) / P.nsplit);
#pragma unroll
    for (int i = 0; i < 2; i++) { k.a[i] = max(k.a[i], k.A); k.b[i] = max(k.a[i], min(k.b[i], k.B)); }
    return k;
  };
  // a step that not every row of the block sees whole
  auto partial = [&](const Walk& k, int j) {
    return j * 128 < k.lo || j * 128 + 128 > k.hi || (P.causal && j * 128 + 127 > k.p_low) || (P.window && j * 128 <= k.p_high - P.window);
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

  if (warp < 8) {
    // ------------------------------------------------------------------------------------------ softmax: a thread a row
    set_regs<true, 184>();
    const int tile = warp >> 2, e = warp & 3, r = e * 32 + lane;
    uint32_t done = 0;                                           // steps of this tile so far: phases of its barriers
    for (int pair = npair - 1 - turn; pair >= 0; pair -= P.tiles) {
      const Walk k = walk(pair);
      const int rr = (pair * 2 + tile) * 128 + r, t = (int)P.group.quot(rr);
      const bool on = t < ch.n;
      const int pos = ch.p0 + (on ? t : ch.n - 1), head = kvh * group + rr - t * group;
      {                                                          // the row of Q, its sign turned if scores are scaled by a negative number
        const uint32_t flip = P.flip ? 0x80008000u : 0u;
        const bf16* src = P.q + (long long)(ch.s + t) * P.q_row + (long long)head * P.q_head;
        unsigned char* dst = smem + F::Q_AT + tile * F::TILE;
#pragma unroll
        for (int q = 0; q < D / 8; q++) {
          uint4 u = on ? reinterpret_cast<const uint4*>(src)[q] : make_uint4(0, 0, 0, 0);
          u.x ^= flip; u.y ^= flip; u.z ^= flip; u.w ^= flip;
          *reinterpret_cast<uint4*>(dst + tile_at(r, q)) = u;
        }
        fence_proxy_async();
        attn_tc::warp_arrive(smem_u32(&ct.q_full));
      }
      const uint32_t tl = tmem + ((uint32_t)(e * 32) << 16), ts = tl + tile * 128, to = tl + 256 + tile * D;
      float m = -INFINITY, l = 0.f;
      const int n = k.b[tile] - k.a[tile];
      for (int c = 0; c < n; c++) {
        const int j = k.a[tile] + c, k0 = j * 128;
        ok = wait_for(smem_u32(&ct.s_full[tile]), (done + c) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        // Half of the scores at a time: all 128 beside what else a thread keeps do not fit its registers. The second half stays there from the search of the maximum,
        // the first is read again; probabilities go over the second, which by then has been read.
        uint32_t s[2][32];
        const uint4 vw = *reinterpret_cast<const uint4*>(ct.valid[j % F::NV]);
        const bool mask = partial(k, j) || (vw.x & vw.y & vw.z & vw.w) != 0xffffffffu;
        auto read = [&](int half) {
          attn_tc::tmem_ld32_nw(ts + half * 64, s[0]);
          attn_tc::tmem_ld32_nw(ts + half * 64 + 32, s[1]);
          attn_tc::tmem_ld_wait();
          if (mask) {
            const int x1 = (P.causal ? pos - k0 : 127) - half * 64, x0 = (P.window ? pos - P.window + 1 - k0 : 0) - half * 64;
            const uint32_t w[2] = {half ? vw.z : vw.x, half ? vw.w : vw.y};
#pragma unroll
            for (int q = 0; q < 2; q++)
#pragma unroll
              for (int x = 0; x < 32; x++)
                if (!((w[q] >> x) & 1) || q * 32 + x > x1 || q * 32 + x < x0) s[q][x] = 0xff800000u;
          }
        };
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int half = 0; half < 2; half++) {
          read(half);
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            mx[x & 2] = attn_tc::max3(mx[x & 2], __uint_as_float(s[0][x]), __uint_as_float(s[0][x + 1]));
            mx[(x & 2) + 1] = attn_tc::max3(mx[(x & 2) + 1], __uint_as_float(s[1][x]), __uint_as_float(s[1][x + 1]));
          }
        }
        const float m_true = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * P.scale_log2);
        if (c == 0) m = m_true;
        else {
          const bool grow = m_true > m + attn_tc::RESCALE_LOG2;
          if (__any_sync(0xffffffffu, grow)) {
            const float alpha = grow ? ex2_approx(m - m_true) : 1.f;
            if (grow) { m = m_true; l *= alpha; }
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
        const u64 sc2 = attn_tc::f2(P.scale_log2, P.scale_log2), nm2 = attn_tc::f2(-ref, -ref);
        u64 sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int half = 1; half >= 0; half--) {
          if (half == 0) read(0);
#pragma unroll
          for (int q = 0; q < 2; q++) {
            uint32_t pk[16];
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const float2 v = attn_tc::unf2(attn_tc::fma2(attn_tc::f2(__uint_as_float(s[q][x]), __uint_as_float(s[q][x + 1])), sc2, nm2));
              const float p0 = ex2_approx(v.x), p1 = ex2_approx(v.y);
              sum[(x >> 1) & 3] = attn_tc::add2(sum[(x >> 1) & 3], attn_tc::f2(p0, p1));
              pk[x >> 1] = pack2f(p0, p1);                       // rounded to bf16 for the product; the sum is taken before
            }
            attn_tc::tmem_st16(ts + 64 + half * 32 + q * 16, pk);
          }
        }
        attn_tc::tmem_st_wait();
        tc_fence_before();
        attn_tc::warp_arrive(smem_u32(&ct.p_full[tile]));
        const float2 s0 = attn_tc::unf2(attn_tc::add2(sum[0], sum[1])), s1 = attn_tc::unf2(attn_tc::add2(sum[2], sum[3]));
        l += (s0.x + s0.y) + (s1.x + s1.y);
      }
      if (ok && n > 0) {
        ok = wait_for(smem_u32(&ct.o_full[tile]), (done + n - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (ok) {                                                  // the row's result, or its part for combine_kernel
        const int olo = *reinterpret_cast<volatile int*>(&ct.odd_lo), ohi = *reinterpret_cast<volatile int*>(&ct.odd_hi);
        const long long g = (long long)(ch.s + t) * P.n_heads + head;
        const float inv = P.nsplit > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
        bf16* dst = P.out + (long long)(ch.s + t) * P.o_row + (long long)head * P.o_head;
        float* part = P.part + (g * P.nsplit + split) * D;
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
              if ((P.causal && key > pos) || (P.window && key <= pos - P.window) || key / 128 < k.a[tile] || key / 128 >= k.b[tile] || !locate(P.b, seq, key, page, at)) continue;
              const char* row = P.c.v + (long long)kvh * P.c.head_b + (long long)page * P.c.page_b + (long long)at * P.c.row_b;
              const int sc = E4M3 ? P.c.vs[(long long)page * P.c.s_page + (long long)kvh * P.c.s_head + (long long)at * P.c.s_row] : 0;
#pragma unroll
              for (int x = 0; x < 32; x++) {
                const float v = held<E4M3>(row, q * 32 + x, sc);
                if (!isfinite(v)) o[x] = __float_as_uint(__uint_as_float(o[x]) + v);
              }
            }
          }
          if (on && P.nsplit == 1) {
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
              float f[8];
#pragma unroll
              for (int y = 0; y < 8; y++) f[y] = __uint_as_float(o[x + y]) * inv;
              *reinterpret_cast<uint4*>(dst + q * 32 + x) = pack8(f);
            }
          } else if (on) {
#pragma unroll
            for (int x = 0; x < 32; x += 4) *reinterpret_cast<uint4*>(part + q * 32 + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
          }
        }
        if (on && P.nsplit > 1) reinterpret_cast<float2*>(P.part + (long long)P.b.n_rows * P.n_heads * P.nsplit * D)[g * P.nsplit + split] = make_float2(m, l);
        else if (on && P.lse) P.lse[g] = l == 0.f ? -INFINITY : m * LN2 + logf(l);
      }
      tc_fence_before();
      done += (uint32_t)n;
      if (!next(ok)) break;
    }
  } else if (warp < 10) {
    // ------------------------------------------------------------------------------------------ products
    set_regs<false, 72>();
    const int tile = warp - 8;
    uint32_t uses = 0, done = 0, round = 0;                      // items through the ring, steps of the tile
    for (int pair = npair - 1 - turn; pair >= 0; pair -= P.tiles) {
      const Walk k = walk(pair);
      if (lane == 0) {
        const uint32_t ts = tmem + tile * 128, to = tmem + 256 + tile * D, sq = base + F::Q_AT + tile * F::TILE;
        constexpr uint32_t I_S = umma_idesc(false, false, 128, 128), I_O = umma_idesc(false, true, 128, D);
        ok = wait_for(smem_u32(&ct.q_full), round & 1);
        uint32_t c = 0;
        for (int j = k.A; j < k.B && ok; j++) {
          const bool mine = j >= k.a[tile] && j < k.b[tile];
#pragma unroll
          for (int half = 0; half < 2; half++) {
            const uint32_t n = uses + 2 * (uint32_t)(j - k.A) + half, slot = n % F::NST;
            const uint32_t sb = base + F::RING_AT + slot * F::TILE;
            ok = ok && wait_for(smem_u32(&ct.full[slot]), (n / F::NST) & 1);
            if (!ok) break;
            if (!mine) { mbar_arrive(smem_u32(&ct.empty[slot])); continue; }
            if (half == 0) {                                     // S = Q K_j^T, into columns whose probabilities the product before has read
              if (c > 0) ok = wait_for(smem_u32(&ct.o_full[tile]), (done + c - 1) & 1);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < D / 16; kk++)
                umma_bf16(ts, umma_smem_desc(sq + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024), umma_smem_desc(sb + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024), I_S, kk > 0 ? 1u : 0u);
              umma_commit(smem_u32(&ct.s_full[tile]));
            } else {                                             // O += P V_j
              ok = wait_for(smem_u32(&ct.p_full[tile]), (done + c) & 1);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < 8; kk++)
                asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                             ::"r"(to), "r"(ts + 64 + kk * 8), "l"(umma_smem_desc(sb + kk * 2048, 16384, 1024)), "r"(I_O), "r"((c > 0 || kk > 0) ? 1u : 0u) : "memory");
              umma_commit(smem_u32(&ct.o_full[tile]));
              c++;
            }
            umma_commit(smem_u32(&ct.empty[slot]));
          }
        }
      }
      uses += 2u * (uint32_t)(k.B - k.A); done += (uint32_t)(k.b[tile] - k.a[tile]); round++;
      if (!next(ok)) break;
    }
  } else {
    // ------------------------------------------------------------------------------------------ loaders
    set_regs<false, 72>();
    constexpr int CH = E4M3 ? D / 16 : D / 8, IT = 16 * CH / 32;      // 16-byte pieces of a held row, of 16 rows for each lane
    constexpr int LAG = E4M3 ? 0 : F::LAG;                       // rows in 8 bits are there when they are written
    const int w = warp - 10;
    uint32_t uses = 0;
    for (int pair = npair - 1 - turn; pair >= 0; pair -= P.tiles) {
      const Walk k = walk(pair);
      const int total = 2 * (k.B - k.A);
      for (int i = 0; i < total + LAG && ok; i++) {
        if (i < total) {
          const uint32_t n = uses + (uint32_t)i, slot = n % F::NST;
          const int j = k.A + (i >> 1);
          const bool is_v = i & 1, part = partial(k, j);
          ok = wait_for(smem_u32(&ct.empty[slot]), ((n / F::NST) & 1) ^ 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          unsigned char* dst = smem + F::RING_AT + slot * F::TILE;
          const uint32_t dst_s = base + F::RING_AT + slot * F::TILE;
          const char* src = (is_v ? P.c.v : P.c.k) + (long long)kvh * P.c.head_b;
          for (int u = (w + F::LOADERS - (i * 8) % F::LOADERS) % F::LOADERS; u < 8; u += F::LOADERS) {
            const int key = j * 128 + u * 16 + (lane & 15);
            int page = 0, at = 0;
            const bool there = key >= k.lo && key < k.hi && locate(P.b, seq, key, page, at);
            const long long off = there ? (long long)page * P.c.page_b + (long long)at * P.c.row_b : -1;
            const uint32_t vb = __ballot_sync(0xffffffffu, there) & 0xffffu;
            if (!is_v && lane == 0) ct.valid[j % F::NV][u] = (uint16_t)vb;
            if (!E4M3 && !part) {
#pragma unroll
              for (int x = 0; x < IT; x++) {
                const int idx = x * 32 + lane, row = idx / CH, q = idx % CH;
                const long long o = __shfl_sync(0xffffffffu, off, row);
                cp16(dst_s + tile_at(u * 16 + row, q), o >= 0 ? src + o + q * 16 : src, o >= 0);
              }
            } else {
              uint32_t f = 0;
              if (E4M3 && there) {
                f = scale_bits((is_v ? P.c.vs : P.c.ks)[(long long)page * P.c.s_page + (long long)kvh * P.c.s_head + (long long)at * P.c.s_row]);
                f |= f << 16;
              }
              bool odd = false;
#pragma unroll
              for (int x0 = 0; x0 < IT; x0 += 4) {
                constexpr int BT = IT < 4 ? IT : 4;
                uint4 v[BT];
#pragma unroll
                for (int x = 0; x < BT; x++) {
                  const int idx = (x0 + x) * 32 + lane, row = idx / CH, q = idx % CH;
                  const long long o = __shfl_sync(0xffffffffu, off, row);
                  v[x] = o >= 0 ? *reinterpret_cast<const uint4*>(src + o + q * 16) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int x = 0; x < BT; x++) {
                  const int idx = (x0 + x) * 32 + lane, row = idx / CH, q = idx % CH;
                  if constexpr (E4M3) {
                    uint32_t fr = __shfl_sync(0xffffffffu, f, row);
                    if (is_v && part && fr == 0x7fc07fc0u) { odd = true; fr = 0; }
                    *reinterpret_cast<uint4*>(dst + tile_at(u * 16 + row, 2 * q)) = make_uint4(widen_lo(v[x].x, fr), widen_hi(v[x].x, fr), widen_lo(v[x].y, fr), widen_hi(v[x].y, fr));
                    *reinterpret_cast<uint4*>(dst + tile_at(u * 16 + row, 2 * q + 1)) = make_uint4(widen_lo(v[x].z, fr), widen_hi(v[x].z, fr), widen_lo(v[x].w, fr), widen_hi(v[x].w, fr));
                  } else {
                    if (is_v && (odd_bits(v[x].x) || odd_bits(v[x].y) || odd_bits(v[x].z) || odd_bits(v[x].w))) {
                      odd = true;
                      v[x] = make_uint4(without_odd(v[x].x), without_odd(v[x].y), without_odd(v[x].z), without_odd(v[x].w));
                    }
                    *reinterpret_cast<uint4*>(dst + tile_at(u * 16 + row, q)) = v[x];
                  }
                }
              }
              if (odd) { atomicMin(&ct.odd_lo, j * 128 + u * 16); atomicMax(&ct.odd_hi, min(k.hi - 1, j * 128 + u * 16 + 15)); }
            }
          }
        }
        cp_commit();
        cp_wait<LAG>();
        if (i >= LAG) {                                       // the copies of the tile LAG before this one have landed: the products may read it
          fence_proxy_async();
          attn_tc::warp_arrive(smem_u32(&ct.full[(uses + (uint32_t)(i - LAG)) % F::NST]));
        }
      }
      cp_wait<0>();
      uses += (uint32_t)total;
      if (!next(ok)) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

}  // namespace paged
}  // namespace ofa
