// Rows of new keys and values to their pages, and back: one pass, bound by its bytes (or, for a step of a few tokens, by one launch and three
// dependent loads: q_start, the page table, the row).
//
// A thread holds 8 values of a row (16 of an 8-bit one: 16 bytes where it is held), so a row is 4 to 16 neighbouring lanes: the largest magnitude is found as an
// unsigned maximum of the bits without signs (an infinity or a NaN is then the largest) and shared by shuffles; scaling by a power of two is exact, so the
// only rounding is the one to e4m3 (to nearest, half a step 2^-4 relative). A block takes consecutive rows of the call; its threads compare the starts of
// all sequences with them once and leave each row's page in shared memory. Two pieces a thread are asked for before the first is worked
// on, in 32 registers, so that an SM holds eight blocks (39,000 rows of 8 heads of 128 out of 8 bits 42.6 us; four pieces and five blocks 45; asking for new rows before their places are
// known, which keeps them in registers meanwhile, 13.2 -> 15.7 for 8,192 rows to 8 bits).
#pragma once
#include <cuda_fp8.h>
#include "paged.cuh"

namespace ofa {
namespace paged {

struct MoveArgs {
  Batch b;
  Pool c;
  bf16 *k, *v;                                        // rows of the call: read by append, written by read
  long long k_row, k_head, v_row, v_head;             // strides in elements
  int n_kv_heads, rows;                               // rows a block takes
  Div pair;                                           // by 2 * n_kv_heads
};
constexpr int MOVE_ROWS = 64;                         // at most

__device__ __forceinline__ uint32_t to_e4m3(uint32_t lo, uint32_t hi, float f) {
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&lo)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&hi));
  const uint32_t x = __nv_cvt_float2_to_fp8x2(make_float2(a.x * f, a.y * f), __NV_SATFINITE, __NV_E4M3);
  const uint32_t y = __nv_cvt_float2_to_fp8x2(make_float2(b.x * f, b.y * f), __NV_SATFINITE, __NV_E4M3);
  return x | y << 16;
}

template <int D, bool E4M3, bool READ>
__global__ void __launch_bounds__(256, 8) move_kernel(const __grid_constant__ MoveArgs P) {
  constexpr int PIECE = E4M3 ? 16 : 8, LANES = D / PIECE;      // values a thread holds of a row, lanes of a row
  after_the_kernel_before();
  __shared__ int2 place[MOVE_ROWS];                   // page and row in it; x = -1: nowhere, -2: no sequence's row
  const int tid = threadIdx.x, r0 = blockIdx.x * P.rows, r1 = min(r0 + P.rows, P.b.n_rows);
  if (tid < MOVE_ROWS) place[tid] = make_int2(-2, 0);
  __syncthreads();
  for (int i = tid; i < P.b.n_seqs; i += 256) {       // the sequence of each row
    const int s = __ldg(P.b.q_start + i), e = __ldg(P.b.q_start + i + 1);
    if (s < 0 || e < s || e > P.b.n_rows) { flag(P.b.status, ST_ROWS); continue; }
    for (int row = max(s, r0); row < min(e, r1); row++) place[row - r0].x = i;
  }
  __syncthreads();
  if (tid < MOVE_ROWS && place[tid].x >= 0) {
    const int i = place[tid].x;
    const Chunk ch = chunk_of(P.b, i);
    const int pos = ch.p0 + (r0 + tid - ch.s);
    int page, at;
    if (!READ && pos < 0 && ch.len > 0) flag(P.b.status, ST_LENGTH);           // a row is lost, unless the sequence is a place in a batch that nobody uses; one that is read is zeros
    if (pos < 0 || !locate(P.b, i, pos, page, at)) page = -1, at = 0;
    place[tid] = make_int2(page, at);
  }
  __syncthreads();
  constexpr int U = 2;                                // pieces that a thread has on their way
  const int total = (r1 - r0) * 2 * P.n_kv_heads * LANES;
  for (int base = 0; base < total; base += 256 * U) {
    bf16* x[U];
    char* held[U];
    unsigned char* sc[U];
    int state[U];                                     // -2 no row, -1 a row without a place, 0 a row with one
    uint4 a[U], b[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int it = base + i * 256 + tid, part = it % LANES, vec = it / LANES, row = (int)P.pair.quot(vec), wh = vec - row * 2 * P.n_kv_heads;
      const bool is_v = wh >= P.n_kv_heads;
      const int head = is_v ? wh - P.n_kv_heads : wh;
      const int2 pl = it < total ? place[row] : make_int2(-2, 0);
      state[i] = min(pl.x, 0);
      x[i] = (is_v ? P.v + (long long)(r0 + row) * P.v_row + (long long)head * P.v_head : P.k + (long long)(r0 + row) * P.k_row + (long long)head * P.k_head) + part * PIECE;
      held[i] = (is_v ? P.c.v : P.c.k) + (long long)pl.x * P.c.page_b + (long long)head * P.c.head_b + (long long)pl.y * P.c.row_b + part * 16;
      if (E4M3) sc[i] = (is_v ? P.c.vs : P.c.ks) + (long long)pl.x * P.c.s_page + (long long)head * P.c.s_head + (long long)pl.y * P.c.s_row;
      a[i] = b[i] = make_uint4(0, 0, 0, 0);           // a row that is nowhere reads as zeros
      if (state[i] == 0) {
        if constexpr (READ) {
          a[i] = *reinterpret_cast<const uint4*>(held[i]);
          if (E4M3) b[i].x = *sc[i];
        } else {
          a[i] = reinterpret_cast<const uint4*>(x[i])[0];
          if (E4M3) b[i] = reinterpret_cast<const uint4*>(x[i])[1];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
      if constexpr (READ) {
        if (state[i] == -2) continue;
        if constexpr (E4M3) {
          uint32_t f = scale_bits((int)b[i].x); f |= f << 16;
          reinterpret_cast<uint4*>(x[i])[0] = make_uint4(widen_lo(a[i].x, f), widen_hi(a[i].x, f), widen_lo(a[i].y, f), widen_hi(a[i].y, f));
          reinterpret_cast<uint4*>(x[i])[1] = make_uint4(widen_lo(a[i].z, f), widen_hi(a[i].z, f), widen_lo(a[i].w, f), widen_hi(a[i].w, f));
        } else *reinterpret_cast<uint4*>(x[i]) = a[i];
      } else if constexpr (E4M3) {
        unsigned m = max(max_bits(a[i]), max_bits(b[i]));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int s = scale_byte(m);
        const float f = __uint_as_float((uint32_t)(254 - (s == SCALE_NAN ? 127 : s)) << 23);          // 2^(127 - s)
        if (state[i] == 0) {
          *reinterpret_cast<uint4*>(held[i]) = s == SCALE_NAN ? make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu)
                                                              : make_uint4(to_e4m3(a[i].x, a[i].y, f), to_e4m3(a[i].z, a[i].w, f), to_e4m3(b[i].x, b[i].y, f), to_e4m3(b[i].z, b[i].w, f));
          if (tid % LANES == 0) *sc[i] = (unsigned char)s;
        }
      } else if (state[i] == 0) *reinterpret_cast<uint4*>(held[i]) = a[i];
    }
  }
}

}  // namespace paged
}  // namespace ofa
