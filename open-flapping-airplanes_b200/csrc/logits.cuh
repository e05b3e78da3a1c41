// What is done to a row of logits before a token is chosen from it, in one pass over the row:
//   x = seen ? (x > 0 ? x / r : x * r) : x         r = repetition[row]; seen: the token stands anywhere in the row's history
//   x = x - frequency[row] * n - presence[row] * (n > 0)       n = how often it stands behind the prompt
//   x = x + sum of the row's biases with this id
//   x = -inf where the mask's bit is 0
// In fp32 whatever the logits' type, rounded once. Bound by reading and writing the logits.
//
// A block takes a stretch of one row's vocabulary and keeps counts and biases of that stretch in shared memory, so the history needs no sort
// and no pass over [rows][vocab] counters: every block reads its row's whole history (from L2 after the first) and counts what falls into its stretch with integer
// atomics, whose order does not matter. A bias that names an id twice is summed in the order of the list by the thread that meets it first.
#pragma once
#include "common.cuh"

namespace ofa {
namespace logits {

struct Args {
  const void* in; void* out;
  long long in_row, out_row;
  int vocab, stretch;                                  // stretch: tokens per block
  const int* tokens; long long tokens_row; int max_tokens;
  const int *n_tokens, *n_prompt;
  const float *repetition, *presence, *frequency;
  const int* bias_ids; const float* bias; long long bias_row; int max_bias;
  const unsigned* mask; long long mask_row;
};
constexpr unsigned PROMPT = 1u << 31;                  // count word: bit 31 = in the prompt, the rest counts the others

template <class T, bool WIDE>
__global__ void __launch_bounds__(256) process_kernel(const __grid_constant__ Args P) {
  constexpr int VN = WIDE ? Vec<T>::N : 1;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned* count = reinterpret_cast<unsigned*>(smem);
  float* add = reinterpret_cast<float*>(smem + (P.tokens ? (size_t)P.stretch * 4 : 0));
  const int tid = threadIdx.x, row = blockIdx.y, v0 = blockIdx.x * P.stretch, nv = min(P.stretch, P.vocab - v0);
  if (P.tokens) {
    for (int i = tid; i < nv; i += 256) count[i] = 0;
  }
  if (P.bias_ids) {
    for (int i = tid; i < nv; i += 256) add[i] = 0.f;
  }
  if (P.tokens || P.bias_ids) __syncthreads();
  if (P.tokens) {
    const int n = P.n_tokens ? min(max(__ldg(P.n_tokens + row), 0), P.max_tokens) : P.max_tokens, first = P.n_prompt ? __ldg(P.n_prompt + row) : 0;
    const int* t = P.tokens + (long long)row * P.tokens_row;
    for (int i = tid; i < n; i += 256) {
      const unsigned at = (unsigned)__ldg(t + i) - (unsigned)v0;
      if (at < (unsigned)nv) { if (i < first) atomicOr(&count[at], PROMPT); else atomicAdd(&count[at], 1u); }
    }
  }
  if (P.bias_ids) {
    const int* ids = P.bias_ids + (long long)row * P.bias_row;
    const float* val = P.bias + (long long)row * P.bias_row;
    for (int i = tid; i < P.max_bias; i += 256) {
      const int id = __ldg(ids + i);
      const unsigned at = (unsigned)id - (unsigned)v0;
      if (id < 0 || at >= (unsigned)nv) continue;
      bool head = true;
      for (int j = 0; j < i && head; j++) head = __ldg(ids + j) != id;
      if (!head) continue;
      float s = __ldg(val + i);
      for (int j = i + 1; j < P.max_bias; j++) if (__ldg(ids + j) == id) s += __ldg(val + j);
      add[at] = s;
    }
  }
  if (P.tokens || P.bias_ids) __syncthreads();
  const float rep = P.repetition ? __ldg(P.repetition + row) : 1.f, pres = P.presence ? __ldg(P.presence + row) : 0.f, freq = P.frequency ? __ldg(P.frequency + row) : 0.f;
  const T* in = reinterpret_cast<const T*>(P.in) + (long long)row * P.in_row + v0;
  T* out = reinterpret_cast<T*>(P.out) + (long long)row * P.out_row + v0;
  const unsigned* mask = P.mask ? P.mask + (long long)row * P.mask_row : nullptr;
  auto one = [&](float x, int i) {
    if (P.tokens) {
      const unsigned n = count[i];
      if (n) {
        x = x > 0.f ? x / rep : x * rep;
        const unsigned made = n & ~PROMPT;
        if (made) x = x - freq * (float)made - pres;
      }
    }
    if (P.bias_ids) x += add[i];
    if (mask && !(__ldg(mask + ((v0 + i) >> 5)) >> ((v0 + i) & 31) & 1)) x = -INFINITY;
    return x;
  };
  for (int i = tid * VN; i < nv; i += 256 * VN) {
    if (VN > 1 && i + VN <= nv) {
      float f[VN];
      if constexpr (VN > 1) {
        ldv(in + i, f);
#pragma unroll
        for (int e = 0; e < VN; e++) f[e] = one(f[e], i + e);
        stv(out + i, f);
      }
    } else {
      for (int e = i; e < min(i + VN, nv); e++) out[e] = from_f<T>(one(to_f(in[e]), e));
    }
  }
}

}  // namespace logits
}  // namespace ofa
