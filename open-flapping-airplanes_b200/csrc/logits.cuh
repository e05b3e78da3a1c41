// What is done to a row of logits before a token is chosen from it, in one pass over the row:
//   x = seen ? (x > 0 ? x / r : x * r) : x         r = repetition[row]; seen: the token stands anywhere in the row's history
//   x = x - frequency[row] * n - presence[row] * (n > 0)       n = how often it stands behind the prompt
//   x = x + sum of the row's biases with this id
//   x = -inf where the mask's bit is 0
// In fp32 whatever the logits' type, rounded once. Bound by reading and writing the logits.
//
// Every stretch of a row needs its own tokens' counts, of the row's whole history. Two ways:
//   process_kernel alone: a block streams a stretch of one row's vocabulary through with the mask, and then changes those few logits that the history or a bias names: it reads the
//     row's whole history (from L2 after the first block), counts what falls into its stretch in a word for each token in shared memory (integer atomics, whose order does
//     not matter) and puts who makes a token's word other than 0 on a list, whose tokens are finished from what the stream left in their places (where the list is
//     too short, by a second look at the history). One launch, for calls of few rows: 4 rows of 50,304 fp32 in 3.0 us.
//   process_kernel for the stream and mask, touch_kernel for the named logits: a block a row counts the history in a hash table of shared memory, large enough for every entry to be
//     another token, while the last blocks of the stream still run. For calls that fill the machine, whose stream is then free of counters: 192 rows of 100,352 bf16 up to 2,000
//     tokens each take 30 us the first way, 21.5 this way, the stream alone 15. What is left are the named logits' sectors, which go to memory twice. (Looking at a token's word for
//     every logit, with the arithmetic of a hit inlined 32 times, took 47.)
// A bias marks its token's word; the entries of its list are added in their order: by process_kernel in shared memory, in one pass over the list; in touch_kernel by each thread with one of them,
// who looks through the list. That is quadratic, so lists of more than 128 take the first way whatever the call's size (192 rows of 100,352 bf16 with 96 biases 22.5 us, the first way 27.8; with
// 160 35.4 and 32.4; with 5,000 8,680 and 260). Stretches begin where a row's 16-byte vectors do, so a row that starts between two boundaries
// loses only its first and last vector to single elements.
#pragma once
#include "paged.cuh"

namespace ofa {
namespace logits {
using paged::after_the_kernel_before;

struct Args {
  const void* in; void* out;
  long long in_row, out_row;
  int vocab;
  const int* tokens; long long tokens_row; int max_tokens;
  const int *n_tokens, *n_prompt;
  const float *repetition, *presence, *frequency;
  const int* bias_ids; const float* bias; long long bias_row; int max_bias;
  const unsigned* mask; long long mask_row;
  int slots_log2;                                              // touch_kernel: of its table
};
constexpr int LISTED = 1024, SHORT_LIST = 128;
enum { STREAM, WORDS, SUMS };                                   // process_kernel: the stream alone; the history's logits too; and the biases'
constexpr unsigned PROMPT = 1u << 31, BIASED = 1u << 30;      // a token's word: in the prompt, has a bias; the rest counts where it stands behind the prompt

// A named token's logit with its word c and the sum of its biases
struct Row { float rep, pres, freq; const int* ids; const float* val; };
__device__ __forceinline__ Row row_of(const Args& P, int row) {
  return {P.repetition ? __ldg(P.repetition + row) : 1.f, P.presence ? __ldg(P.presence + row) : 0.f, P.frequency ? __ldg(P.frequency + row) : 0.f,
          P.bias_ids + (long long)row * P.bias_row, P.bias + (long long)row * P.bias_row};
}
__device__ __forceinline__ float bias_of(const Args& P, const Row& R, int t) {
  float s = 0.f;
#pragma unroll 4
  for (int j = 0; j < P.max_bias; j++) if (__ldg(R.ids + j) == t) s += __ldg(R.val + j);
  return s;
}
__device__ __forceinline__ float touched(const Row& R, float f, unsigned c, float bias) {
  const unsigned made = c & ~(PROMPT | BIASED);
  if (made || (c & PROMPT)) f = f > 0.f ? f / R.rep : f * R.rep;
  if (made) f = f - R.freq * (float)made - R.pres;
  return c & BIASED ? f + bias : f;
}

template <class T, int VECS, bool WIDE, int MODE>
__global__ void __launch_bounds__(256) process_kernel(const __grid_constant__ Args P) {
  constexpr int VN = Vec<T>::N, S = 256 * VN * VECS;           // tokens of a block
  after_the_kernel_before();
  extern __shared__ __align__(16) unsigned count[];
  __shared__ int list[LISTED], listed;
  const int tid = threadIdx.x, row = blockIdx.y;
  const T* in = reinterpret_cast<const T*>(P.in) + (long long)row * P.in_row;
  T* out = reinterpret_cast<T*>(P.out) + (long long)row * P.out_row;
  const int v0 = (int)blockIdx.x * S - (WIDE ? (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T)) : 0);
  const bool words = MODE == SUMS || (MODE == WORDS && P.tokens);
  float* sums = reinterpret_cast<float*>(count + S);           // SUMS: by token of the stretch
  if (MODE == STREAM) cudaTriggerProgrammaticLaunchCompletion();       // touch_kernel may begin to count
  uint4 x[VECS];
#pragma unroll
  for (int k = 0; k < VECS; k++) {
    const int t = v0 + (k * 256 + tid) * VN;
    if (WIDE && t >= 0 && t + VN <= P.vocab) x[k] = *reinterpret_cast<const uint4*>(in + t);
  }
  const unsigned* mask = P.mask ? P.mask + (long long)row * P.mask_row : nullptr;
  const int* ids = P.bias_ids + (long long)row * P.bias_row;
  const int* text = P.tokens + (long long)row * P.tokens_row;
  int n = 0;
  // a token's word, nullptr for one that is not of this stretch
  auto word = [&](int id) {
    const unsigned at = (unsigned)id - (unsigned)v0;
    return (unsigned)id < (unsigned)P.vocab && at < (unsigned)S ? count + at : nullptr;
  };
  auto put = [&](int t) { const int at = atomicAdd(&listed, 1); if (at < LISTED) list[at] = t; };
  if (words) {
#pragma unroll
    for (int i = 0; i < S / 1024 * (MODE == SUMS ? 2 : 1); i++) reinterpret_cast<uint4*>(count)[i * 256 + tid] = make_uint4(0, 0, 0, 0);
    if (tid == 0) listed = 0;
    __syncthreads();
    if (P.tokens) {
      n = P.n_tokens ? min(max(__ldg(P.n_tokens + row), 0), P.max_tokens) : P.max_tokens;
      const int first = P.n_prompt ? __ldg(P.n_prompt + row) : 0;
      for (int base = tid; base < P.max_tokens; base += 1024) {
        int t[4];                                              // asked for side by side, and without waiting for how many count
#pragma unroll
        for (int u = 0; u < 4; u++) t[u] = base + u * 256 < P.max_tokens ? __ldg(text + base + u * 256) : -1;
        if (base >= n) break;
#pragma unroll
        for (int u = 0; u < 4; u++) {
          unsigned* w = base + u * 256 < n ? word(t[u]) : nullptr;
          if (w && (base + u * 256 < first ? atomicOr(w, PROMPT) : atomicAdd(w, 1u)) == 0) put(t[u]);
        }
      }
    }
    if constexpr (MODE == SUMS) {
      // A warp sums the tokens of every eighth place, so that a token's entries are added by one warp, in the order of the list: 32 entries at once, the same token's in turns
      const int lane = tid & 31, warp = tid >> 5;
      const float* val = P.bias + (long long)row * P.bias_row;
#pragma unroll 1
      for (int base = lane; base - lane < P.max_bias; base += 128) {
        int t[4];
#pragma unroll
        for (int u = 0; u < 4; u++) t[u] = base + u * 32 < P.max_bias ? __ldg(ids + base + u * 32) : -1;
#pragma unroll
        for (int u = 0; u < 4; u++) {
          unsigned* w = word(t[u]);
          const int at = w ? (int)(w - count) : -1;
          const bool mine = w && (at & 7) == warp;
          if (!__any_sync(0xffffffffu, mine)) continue;
          const float v = mine ? __ldg(val + base + u * 32) : 0.f;
          const int turn = __popc(__match_any_sync(0xffffffffu, mine ? at : -1) & ((1u << lane) - 1)), turns = (int)__reduce_max_sync(0xffffffffu, mine ? turn : 0);
          if (mine && turn == 0 && atomicOr(w, BIASED) == 0) put(t[u]);
          for (int i = 0; i <= turns; i++) {
            if (mine && turn == i) sums[at] += v;
            __syncwarp();
          }
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < VECS; k++) {
    const int at = (k * 256 + tid) * VN, t = v0 + at;
    if (WIDE && t >= 0 && t + VN <= P.vocab) {
      if (mask) {
        const unsigned lo = __ldg(mask + (t >> 5)), hi = (t & 31) + VN > 32 ? __ldg(mask + (t >> 5) + 1) : 0u;
        const unsigned bits = __funnelshift_r(lo, hi, t & 31);
        float f[VN];
        ldv(reinterpret_cast<const T*>(&x[k]), f);
#pragma unroll
        for (int e = 0; e < VN; e++) if (!(bits >> e & 1)) f[e] = -INFINITY;
        stv(out + t, f);
      } else *reinterpret_cast<uint4*>(out + t) = x[k];
    } else {
#pragma unroll 1
      for (int e = 0; e < VN; e++) {                           // single elements: side by side over the threads where no vector is whole
        const int t1 = v0 + (WIDE ? at + e : k * 256 * VN + e * 256 + tid);
        if (t1 >= 0 && t1 < P.vocab) out[t1] = !mask || (__ldg(mask + (t1 >> 5)) >> (t1 & 31) & 1) ? in[t1] : from_f<T>(-INFINITY);
      }
    }
  }
  if (!words) return;
  __syncthreads();
  const Row R = row_of(P, row);
  const bool all = listed <= LISTED;
#pragma unroll 1
  for (int i = tid; i < (all ? listed : n + (MODE == SUMS ? P.max_bias : 0)); i += 256) {
    const int t = all ? list[i] : i < n ? __ldg(text + i) : __ldg(ids + i - n);
    unsigned* w = word(t);
    const unsigned c = w ? atomicExch(w, 0u) : 0u;
    if (!c || (mask && !(__ldg(mask + (t >> 5)) >> (t & 31) & 1))) continue;
    out[t] = from_f<T>(touched(R, to_f(out[t]), c, MODE == SUMS && (c & BIASED) ? sums[w - count] : 0.f));
  }
}

// The named logits of a row, behind the stream. The table holds a token + 1, its word and the sum of its biases, which each thread with one of them forms (the same
// value). With a quarter of the slots in use few lanes probe twice; at a half a warp's longest chain of atomics took 6 us. All that needs only the tokens is
// asked for side by side, before it is known how many count and while the stream still runs.
template <class T> __global__ void __launch_bounds__(512) touch_kernel(const __grid_constant__ Args P) {
  extern __shared__ __align__(16) unsigned table[];
  const int tid = threadIdx.x, row = blockIdx.x, slots = 1 << P.slots_log2, most = P.tokens ? P.max_tokens : 0, named = most + P.max_bias;
  unsigned *keys = table, *words = table + slots;
  float* sums = reinterpret_cast<float*>(words + slots);
  const T* in = reinterpret_cast<const T*>(P.in) + (long long)row * P.in_row;
  T* out = reinterpret_cast<T*>(P.out) + (long long)row * P.out_row;
  const unsigned* mask = P.mask ? P.mask + (long long)row * P.mask_row : nullptr;
  const int* text = P.tokens + (long long)row * P.tokens_row;
  const Row R = row_of(P, row);
  const int n = !P.tokens ? 0 : P.n_tokens ? __ldg(P.n_tokens + row) : most, first = P.tokens && P.n_prompt ? __ldg(P.n_prompt + row) : 0;
  constexpr int U = 4;                                         // entries of a thread: of the history, then the biases
  int t[U];
  T x[U];
  unsigned allowed[U];
  auto ask = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = base + u * 512;
      t[u] = i < most ? __ldg(text + i) : i < named ? __ldg(R.ids + i - most) : -1;
      if ((unsigned)t[u] >= (unsigned)P.vocab || (i < most && i >= n)) t[u] = -1;
    }
  };
  auto count = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (t[u] < 0) continue;
      const int i = base + u * 512;
      unsigned at = (unsigned)t[u] * 2654435769u >> (32 - P.slots_log2);        // Fibonacci hashing
      while (true) {                                           // ends: there are more slots than entries
        const unsigned was = atomicCAS(keys + at, 0u, (unsigned)t[u] + 1);
        if (was == 0 || was == (unsigned)t[u] + 1) break;
        at = (at + 1) & (slots - 1);
      }
      if (i >= most) { sums[at] = bias_of(P, R, t[u]); atomicOr(words + at, BIASED); }
      else if (i < first) atomicOr(words + at, PROMPT);
      else atomicAdd(words + at, 1u);
    }
  };
  auto look = [&] {                                            // the logits as they came: in place the stream writes back what it read
#pragma unroll
    for (int u = 0; u < U; u++) {
      allowed[u] = t[u] < 0 ? 0u : mask ? __ldg(mask + (t[u] >> 5)) >> (t[u] & 31) : 1u;
      x[u] = in[max(t[u], 0)];
    }
  };
  auto finish = [&] {                                          // by the first thread that comes for a token
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (!(allowed[u] & 1)) continue;
      unsigned at = (unsigned)t[u] * 2654435769u >> (32 - P.slots_log2);
      while (keys[at] != (unsigned)t[u] + 1) at = (at + 1) & (slots - 1);      // it is there
      if (const unsigned c = atomicExch(words + at, 0u)) out[t[u]] = from_f<T>(touched(R, to_f(x[u]), c, sums[at]));
    }
  };
  ask(tid);
  for (int i = tid; i < slots / 2; i += 512) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (named > 512 * U)
    for (int base = tid + 512 * U; base < named; base += 512 * U) { ask(base); count(base); }
  if (named > 512 * U) ask(tid);
  look();
  count(tid);
  __syncthreads();
  cudaGridDependencySynchronize();
  finish();
  if (named > 512 * U)
    for (int base = tid + 512 * U; base < named; base += 512 * U) { ask(base); look(); finish(); }
}

}  // namespace logits
}  // namespace ofa
