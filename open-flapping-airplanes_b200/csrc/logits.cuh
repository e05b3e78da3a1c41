// What is done to a row of logits before a token is chosen from it, in one pass over the row:
//   x = seen ? (x > 0 ? x / r : x * r) : x         r = repetition[row]; seen: the token stands anywhere in the row's history
//   x = x - frequency[row] * n - presence[row] * (n > 0)       n = how often it stands behind the prompt
//   x = x + sum of the row's biases with this id
//   x = -inf where the mask's bit is 0
// In fp32 whatever the logits' type, rounded once. Bound by reading and writing the logits.
//
// A block takes a stretch of one row's vocabulary and keeps a word for each of its tokens in shared memory, so the history needs no sort
// and no pass over [rows][vocab] counters: every block reads its row's whole history (from L2 after the first) and counts what falls into its stretch with integer
// atomics, whose order does not matter; a bias marks its token, and the few threads that meet a mark add the list's entries for it in their order. The logits are asked for before
// all that. Stretches begin where a row's 16-byte vectors do, so a row that starts between two boundaries loses only its first and last vector to single elements.
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
constexpr unsigned PROMPT = 1u << 31, BIASED = 1u << 30;      // a token's word: in the prompt, has a bias; the rest counts where it stands behind the prompt

template <class T, int VECS, bool WIDE>
__global__ void __launch_bounds__(256) process_kernel(const __grid_constant__ Args P) {
  constexpr int VN = Vec<T>::N, S = 256 * VN * VECS;           // tokens of a block
  extern __shared__ __align__(16) unsigned count[];
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
  const float rep = P.repetition ? __ldg(P.repetition + row) : 1.f, pres = P.presence ? __ldg(P.presence + row) : 0.f, freq = P.frequency ? __ldg(P.frequency + row) : 0.f;
  const unsigned* mask = P.mask ? P.mask + (long long)row * P.mask_row : nullptr;
  const int* ids = P.bias_ids + (long long)row * P.bias_row;
  const float* val = P.bias + (long long)row * P.bias_row;
  if (words) {
#pragma unroll
    for (int i = 0; i < S / 1024; i++) reinterpret_cast<uint4*>(count)[i * 256 + tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (P.tokens) {
      const int n = P.n_tokens ? min(max(__ldg(P.n_tokens + row), 0), P.max_tokens) : P.max_tokens, first = P.n_prompt ? __ldg(P.n_prompt + row) : 0;
      const int* t = P.tokens + (long long)row * P.tokens_row;
#pragma unroll 4
      for (int i = tid; i < n; i += 256) {
        const int id = __ldg(t + i);
        const unsigned at = (unsigned)id - (unsigned)v0;
        if ((unsigned)id < (unsigned)P.vocab && at < (unsigned)S) { if (i < first) atomicOr(&count[at], PROMPT); else atomicAdd(&count[at], 1u); }
      }
    }
    if (P.bias_ids) {
      for (int i = tid; i < P.max_bias; i += 256) {
        const int id = __ldg(ids + i);
        const unsigned at = (unsigned)id - (unsigned)v0;
        if ((unsigned)id < (unsigned)P.vocab && at < (unsigned)S) atomicOr(&count[at], BIASED);
      }
    }
    __syncthreads();
  }
  auto one = [&](float f, int t, unsigned n, bool allowed) {   // token t, its word
    if (n) {
      const unsigned made = n & ~(PROMPT | BIASED);
      if (made || (n & PROMPT)) f = f > 0.f ? f / rep : f * rep;
      if (made) f = f - freq * (float)made - pres;
      if (n & BIASED) {
        float s = 0.f;
#pragma unroll 4
        for (int j = 0; j < P.max_bias; j++) if (__ldg(ids + j) == t) s += __ldg(val + j);
        f += s;
      }
    }
    return allowed ? f : -INFINITY;
  };
#pragma unroll
  for (int k = 0; k < VECS; k++) {
    const int at = (k * 256 + tid) * VN, t = v0 + at;
    if (WIDE && t >= 0 && t + VN <= P.vocab) {
      unsigned bits = (1u << VN) - 1;
      if (mask) {
        const unsigned lo = __ldg(mask + (t >> 5)), hi = (t & 31) + VN > 32 ? __ldg(mask + (t >> 5) + 1) : 0u;
        bits = __funnelshift_r(lo, hi, t & 31);
      }
      float f[VN];
      ldv(reinterpret_cast<const T*>(&x[k]), f);
#pragma unroll
      for (int e = 0; e < VN; e += 4) {
        const uint4 n = words ? *reinterpret_cast<const uint4*>(count + at + e) : make_uint4(0, 0, 0, 0);
        f[e] = one(f[e], t + e, n.x, bits >> e & 1); f[e + 1] = one(f[e + 1], t + e + 1, n.y, bits >> (e + 1) & 1);
        f[e + 2] = one(f[e + 2], t + e + 2, n.z, bits >> (e + 2) & 1); f[e + 3] = one(f[e + 3], t + e + 3, n.w, bits >> (e + 3) & 1);
      }
      stv(out + t, f);
    } else {
#pragma unroll 1
      for (int e = 0; e < VN; e++) {                           // single elements: side by side over the threads where no vector is whole
        const int a = WIDE ? at + e : k * 256 * VN + e * 256 + tid, t1 = v0 + a;
        if (t1 >= 0 && t1 < P.vocab) out[t1] = from_f<T>(one(to_f(in[t1]), t1, words ? count[a] : 0u, !mask || (__ldg(mask + (t1 >> 5)) >> (t1 & 31) & 1)));
      }
    }
  }
}

}  // namespace logits
}  // namespace ofa
