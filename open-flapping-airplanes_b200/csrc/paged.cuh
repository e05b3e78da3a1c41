// What the serving operators over a paged key/value cache share: where a position's rows lie, how a row is held in 8 bits, and the
// checks that keep a bad page table or length from becoming a bad access.
//
// A cache is n_pages pages of page_size rows for each key/value head; strides are free, a row's head_dim values lie side by side. Position p of
// sequence i is row p % page_size of page pages[i][p / page_size]. Row t of the n rows that a sequence brings to a call (q_start[i] .. q_start[i + 1])
// has position kv_len[i] - n + t.
//
// 8-bit rows: e4m3 numbers and one byte b for each row and head, standing for code * 2^(b - 127). The scale is a power of two, so that a held value
// is a bf16 number exactly (4 significant bits): reading back rounds nothing, and attention over the cache is attention over those bf16 values.
// A factor amax / 448 would use up to one more binade below and cost a rounding of every value read, or a multiplication of every score and probability.
#pragma once
#include "common.cuh"

namespace ofa {
namespace paged {

enum { ST_PAGE = 1, ST_LENGTH = 2, ST_ROWS = 4, ST_TIMEOUT = 8 };     // bits of the caller's status word

// n / d for 0 <= n < 2^31 (d >= 1): a multiplication instead of a division of 20 instructions
struct Div {
  unsigned d, magic, shift;
  void set(unsigned divisor) {
    d = divisor; shift = 0;
    while ((1ull << shift) < d) shift++;
    magic = (unsigned)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ unsigned quot(unsigned n) const { return (__umulhi(n, magic) + n) >> shift; }
};

struct Batch {
  const int *q_start, *kv_len, *pages;
  long long pages_stride;
  int n_seqs, max_pages, n_pages, n_rows;
  Div page;
  int* status;
};
struct Pool {
  char *k, *v;                                        // pages
  unsigned char *ks, *vs;                             // scale bytes (8-bit rows)
  long long page_b, head_b, row_b;                    // strides of k and v in bytes
  long long s_page, s_head, s_row;                    // strides of ks and vs
};

// The serving kernels are launched as dependents of whatever runs before them in the stream: their launch is then prepared while that still runs, and every block waits here,
// before it touches memory, until it has ended (a block that left without waiting would let the next kernel run ahead of the one before).
__device__ __forceinline__ void after_the_kernel_before() { cudaGridDependencySynchronize(); }

static __device__ __noinline__ void flag(int* status, int bits) { if (status) atomicOr(status, bits); }

// Rows [s, s + n) of the call belong to sequence i, the first of them at position p0 (negative: the sequence is shorter than what it brings).
struct Chunk { int s, n, p0, len; };
__device__ __forceinline__ Chunk chunk_of(const Batch& B, int i) {
  const int s = __ldg(B.q_start + i), e = __ldg(B.q_start + i + 1), len = __ldg(B.kv_len + i);
  if (s < 0 || e < s || e > B.n_rows) { flag(B.status, ST_ROWS); return {0, 0, 0, 0}; }
  if (len < 0) { flag(B.status, ST_LENGTH); return {s, e - s, s - e, 0}; }
  return {s, e - s, len - (e - s), len};
}
// Keys that attention over a context of this length reaches: those that the page table has, at most 2^31 - 1024: what is looked up ahead of a step has a position of 31 bits too
__device__ __forceinline__ int reach(const Batch& B, int len) { return (int)min(min((long long)B.max_pages * B.page.d, 0x7ffffc00ll), (long long)len); }
// page and row of position pos (>= 0) of sequence i; false, and a bit in the status word, where the table has none
__device__ __forceinline__ bool locate(const Batch& B, int i, int pos, int& page, int& at) {
  const unsigned idx = B.page.quot((unsigned)pos);
  if (idx >= (unsigned)B.max_pages) { flag(B.status, ST_LENGTH); return false; }
  page = __ldg(B.pages + (long long)i * B.pages_stride + idx);
  at = pos - (int)(idx * B.page.d);
  if ((unsigned)page >= (unsigned)B.n_pages) { flag(B.status, ST_PAGE); return false; }
  return true;
}

// ---------------------------------------------------------------------------------------------- rows in 8 bits
// Scale byte 255: a row that held an infinity or a NaN, it reads back as NaN. Others are 27 .. 134 (2^-100 .. 2^7): every code times its scale is
// then a normal bf16 number or zero, and 2^120 times the scale (below) fits bf16.
constexpr int SCALE_NAN = 255, E_MIN = -100, E_MAX = 7;

// scale byte for a row whose largest magnitude has these bf16 bits: the smallest power of two by which it fits 448 = 1.75 * 2^8
__device__ __forceinline__ int scale_byte(unsigned amax_bits) {
  if (amax_bits >= 0x7f80u) return SCALE_NAN;
  const int e = (int)(amax_bits >> 7) - 127 - 8 + ((amax_bits & 0x7f) > 0x60 ? 1 : 0);
  return min(max(e, E_MIN), E_MAX) + 127;
}
// The bits of an e4m3 number, moved to where bf16 has sign, exponent and mantissa, are 2^-120 times its value (subnormals too); this is 2^120 times the
// scale, as bf16 bits. One multiplication, exact, then gives the held value.
__device__ __forceinline__ uint32_t scale_bits(int b) { return b == SCALE_NAN ? 0x7fc0u : (uint32_t)(min(b, E_MAX + 127) + 120) << 7; }
// the largest magnitude's bits of eight bf16 numbers; an infinity or a NaN is the largest
__device__ __forceinline__ unsigned max_bits(uint4 u) {
  unsigned m = 0;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) m = max(m, max(w[i] & 0x7fffu, w[i] >> 16 & 0x7fffu));
  return m;
}
// Two e4m3 numbers as bf16 of 2^-120 times their codes' values, three instructions. sel places them in bytes 0 and 2 with their signs in the bytes above, so that one shift moves both.
__device__ __forceinline__ uint32_t raw_pair(uint32_t x, uint32_t y, uint32_t sel) {
  uint32_t w;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(w) : "r"(x), "r"(y), "r"(sel));
  return (w << 4) & 0x87f087f0u;
}
__host__ __device__ constexpr uint32_t raw_sel(int a, int b) { return (uint32_t)(a | (8 | a) << 4 | b << 8 | (8 | b) << 12); }      // of bytes a and b of the eight in (x, y)
// elements 0 and 1, or 2 and 3, of the four in w; f holds the scale_bits of each
__device__ __forceinline__ uint32_t scaled(uint32_t t, uint32_t f) { uint32_t r; asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(t), "r"(f)); return r; }
__device__ __forceinline__ uint32_t widen_lo(uint32_t w, uint32_t f) { return scaled(raw_pair(w, w, raw_sel(0, 1)), f); }
__device__ __forceinline__ uint32_t widen_hi(uint32_t w, uint32_t f) { return scaled(raw_pair(w, w, raw_sel(2, 3)), f); }

}  // namespace paged
}  // namespace ofa
