// What is done to a row of logits before a token is chosen from it, in one pass over the row:
//   x = seen ? (x > 0 ? x / r : x * r) : x         r = repetition[row]; seen: the token stands anywhere in the row's history
//   x = x - frequency[row] * n - presence[row] * (n > 0)       n = how often it stands behind the prompt
//   x = x + sum of the row's biases with this id
//   x = -inf where the mask's bit is 0
// In fp32 whatever the logits' type, rounded once. Bound by reading and writing the logits.
//
// A block takes a stretch of one row's vocabulary. It streams the logits through with the mask alone, and then changes those few that the history or a bias names:
// every block reads its row's whole history (from L2 after the first), counts what falls into its stretch in a word for each token in shared memory (integer atomics, whose order does
// not matter; no sort, no pass over [rows][vocab] counters). Who makes a token's word other than 0 puts it on a list, and the listed tokens are finished from what the stream left in their
// places (where the list is too short, by a second look at the history). Looking at a token's word for every logit instead, with the arithmetic of a hit inlined 32 times, took 47 us
// where this takes 29 (192 rows of 100,352 bf16); a second look at the history in every block 31. A bias marks its token's word; the entries of its list are added in their order. Stretches begin where a row's 16-byte vectors do, so a row that starts between two boundaries loses only its first and last vector to single
// elements.
#pragma once
#include "common.cuh"

namespace ofa {
namespace logits {

struct Args {
  const void* in; void* out;
  long long in_row, out_row;
  int vocab;
  const int* tokens; long long tokens_row; int max_tokens;
  const int *n_tokens, *n_prompt;
  const float *repetition, *presence, *frequency;
  const int* bias_ids; const float* bias; long long bias_row; int max_bias;
  const unsigned* mask; long long mask_row;
};
constexpr int LISTED = 1024;
constexpr unsigned PROMPT = 1u << 31, BIASED = 1u << 30;      // a token's word: in the prompt, has a bias; the rest counts where it stands behind the prompt

template <class T, int VECS, bool WIDE>
__global__ void __launch_bounds__(256) process_kernel(const __grid_constant__ Args P) {
  constexpr int VN = Vec<T>::N, S = 256 * VN * VECS;           // tokens of a block
  extern __shared__ __align__(16) unsigned count[];
  __shared__ int list[LISTED], listed;
  const int tid = threadIdx.x, row = blockIdx.y;
  const T* in = reinterpret_cast<const T*>(P.in) + (long long)row * P.in_row;
  T* out = reinterpret_cast<T*>(P.out) + (long long)row * P.out_row;
  const int v0 = (int)blockIdx.x * S - (WIDE ? (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T)) : 0);
  const bool words = P.tokens || P.bias_ids;
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
    for (int i = 0; i < S / 1024; i++) reinterpret_cast<uint4*>(count)[i * 256 + tid] = make_uint4(0, 0, 0, 0);
    if (tid == 0) listed = 0;
    __syncthreads();
    if (P.tokens) {
      n = P.n_tokens ? min(max(__ldg(P.n_tokens + row), 0), P.max_tokens) : P.max_tokens;
      const int first = P.n_prompt ? __ldg(P.n_prompt + row) : 0;
#pragma unroll 4
      for (int i = tid; i < n; i += 256) {
        const int t = __ldg(text + i);
        unsigned* w = word(t);
        if (w && (i < first ? atomicOr(w, PROMPT) : atomicAdd(w, 1u)) == 0) put(t);
      }
    }
    if (P.bias_ids)
      for (int i = tid; i < P.max_bias; i += 256) { const int t = __ldg(ids + i); unsigned* w = word(t); if (w && atomicOr(w, BIASED) == 0) put(t); }
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
  const float* val = P.bias + (long long)row * P.bias_row;
  const float rep = P.repetition ? __ldg(P.repetition + row) : 1.f, pres = P.presence ? __ldg(P.presence + row) : 0.f, freq = P.frequency ? __ldg(P.frequency + row) : 0.f;
  const bool all = listed <= LISTED;
#pragma unroll 1
  for (int i = tid; i < (all ? listed : n + P.max_bias); i += 256) {           // max_bias is 0 without biases
    const int t = all ? list[i] : i < n ? __ldg(text + i) : __ldg(ids + i - n);
    unsigned* w = word(t);
    const unsigned c = w ? atomicExch(w, 0u) : 0u;
    if (!c || (mask && !(__ldg(mask + (t >> 5)) >> (t & 31) & 1))) continue;
    const unsigned made = c & ~(PROMPT | BIASED);
    float f = to_f(out[t]);
    if (made || (c & PROMPT)) f = f > 0.f ? f / rep : f * rep;
    if (made) f = f - freq * (float)made - pres;
    if (c & BIASED) {
      float s = 0.f;
#pragma unroll 4
      for (int j = 0; j < P.max_bias; j++) if (__ldg(ids + j) == t) s += __ldg(val + j);
      f += s;
    }
    out[t] = from_f<T>(f);
  }
}

}  // namespace logits
}  // namespace ofa
