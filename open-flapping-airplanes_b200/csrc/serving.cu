// Serving operators on the caller's stream (include/ofa_b200.h, "serving over a paged cache"): argument checks and launches. They allocate
// nothing, keep nothing from one call to the next and touch no other stream, so they can be captured into graphs and run side by side.
#include "../../include/ofa_b200.h"
#include "logits.cuh"
#include "paged_attn_tc.cuh"
#include "paged_move.cuh"
#include <cuda_runtime.h>
#include <algorithm>
#include <atomic>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>

using namespace ofa;

namespace {

thread_local char g_error[256] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof g_error, fmt, ap);
  va_end(ap);
  return code;
}
int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return OFA_OK;
  cudaGetLastError();                                            // reported here, not by the next call
  return fail(OFA_CUDA_ERROR, "%s: %s", what, cudaGetErrorString(e));
}
bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
// Whether places of `unit` elements at these strides lie upon one another: from the smallest stride up, each has to pass what lies inside it
struct Axis { long long stride, count; };
bool overlap(Axis a, Axis b, Axis c, long long unit, Axis d = {0, 1}) {
  Axis x[4] = {a, b, c, d};
  std::sort(x, x + 4, [](const Axis& u, const Axis& v) { return u.stride < v.stride; });
  for (const Axis& i : x)
    if (i.count > 1) {
      if (i.stride < unit) return true;
      unit += i.stride * (i.count - 1);
    }
  return false;
}

// Whether two sets of such places, which start at p and q and are alike otherwise, lie upon one another: the second is one more axis, as far as it begins inside the longest step of the first
bool twins(Axis a, Axis b, Axis c, long long unit, const void* p, const void* q, long long size) {
  long long d = std::abs((long long)(reinterpret_cast<intptr_t>(p) - reinterpret_cast<intptr_t>(q))) / size, step = 0, end = unit;
  for (const Axis& i : {a, b, c})
    if (i.count > 1) { step = std::max(step, i.stride); end += i.stride * (i.count - 1); }
  return d < end && overlap(a, b, c, unit, {step ? d % step : d, 2});
}

// ---- checks shared by the operators over a cache
int check_cache(const ofa_kv_cache* c, const ofa_kv_batch* b, int n_rows, paged::Batch& B, paged::Pool& C) {
  if (!c || !b) return fail(OFA_BAD_ARGUMENT, "null pointer");
  if (c->dtype != OFA_KV_BF16 && c->dtype != OFA_KV_E4M3) return fail(OFA_BAD_ARGUMENT, "cache dtype %d is neither OFA_KV_BF16 nor OFA_KV_E4M3", c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(OFA_BAD_ARGUMENT, "head_dim %d: 64 and 128 are built", c->head_dim);
  if (c->n_kv_heads < 1 || c->n_kv_heads > 65535) return fail(OFA_BAD_ARGUMENT, "n_kv_heads %d is outside 1 .. 65535", c->n_kv_heads);
  if (c->page_size < 1 || c->n_pages < 0) return fail(OFA_BAD_ARGUMENT, "page_size %d, n_pages %d", c->page_size, c->n_pages);
  if (n_rows < 0 || b->n_seqs < 0 || b->max_pages < 0 || b->max_new < 0 || b->max_kv < 0)
    return fail(OFA_BAD_ARGUMENT, "negative size: n_rows %d, n_seqs %d, max_pages %d, max_new %d, max_kv %d", n_rows, b->n_seqs, b->max_pages, b->max_new, b->max_kv);
  if (n_rows > 0x7fffff00) return fail(OFA_BAD_ARGUMENT, "%d rows are too many for one call", n_rows);
  const bool e4m3 = c->dtype == OFA_KV_E4M3;
  const long long es = e4m3 ? 1 : 2;
  if (n_rows > 0 && b->n_seqs > 0) {
    if (!b->q_start || !b->kv_len || (b->max_pages > 0 && !b->pages)) return fail(OFA_BAD_ARGUMENT, "null pointer in the batch");
    if (c->n_pages > 0 && (!c->k || !c->v)) return fail(OFA_BAD_ARGUMENT, "null pointer in the cache");
    if (e4m3 && c->n_pages > 0 && (!c->k_scale || !c->v_scale)) return fail(OFA_BAD_ARGUMENT, "an e4m3 cache needs scales");
  }
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || (c->page_stride * es) % 16 || (c->head_stride * es) % 16 || (c->row_stride * es) % 16)
    return fail(OFA_BAD_ARGUMENT, "cached rows start on 16-byte boundaries: pointers and strides");
  if (c->page_stride < 0 || c->head_stride < 0 || c->row_stride < 0 || c->scale_page_stride < 0 || c->scale_head_stride < 0 || c->scale_row_stride < 0 || b->pages_stride < 0)
    return fail(OFA_BAD_ARGUMENT, "negative stride");
  if (!aligned(b->q_start, 4) || !aligned(b->kv_len, 4) || !aligned(b->pages, 4) || !aligned(b->status, 4)) return fail(OFA_BAD_ARGUMENT, "misaligned index array");
  B.q_start = b->q_start; B.kv_len = b->kv_len; B.pages = b->pages; B.pages_stride = b->pages_stride;
  B.n_seqs = b->n_seqs; B.max_pages = b->max_pages; B.n_pages = c->n_pages; B.n_rows = n_rows; B.page.set((unsigned)c->page_size); B.status = b->status;
  C.k = static_cast<char*>(c->k); C.v = static_cast<char*>(c->v); C.ks = c->k_scale; C.vs = c->v_scale;
  C.page_b = c->page_stride * es; C.head_b = c->head_stride * es; C.row_b = c->row_stride * es;
  C.s_page = c->scale_page_stride; C.s_head = c->scale_head_stride; C.s_row = c->scale_row_stride;
  return OFA_OK;
}
int check_rows(const char* name, const void* p, Axis row, Axis head, int dim, bool written) {
  if (!p) return fail(OFA_BAD_ARGUMENT, "%s is null", name);
  if (!aligned(p, 16) || row.stride % 8 || head.stride % 8 || row.stride < 0 || head.stride < 0) return fail(OFA_BAD_ARGUMENT, "rows of %s start on 16-byte boundaries: pointer and strides", name);
  if (written && overlap(row, head, {0, 1}, dim)) return fail(OFA_BAD_ARGUMENT, "rows of %s overlap: strides %lld and %lld", name, row.stride, head.stride);
  return OFA_OK;
}

// The limit of dynamic shared memory, raised once for each kernel and device to all a block may have beside the kernel's own
template <auto KERNEL> cudaError_t allow() {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return e;
  cudaFuncAttributes own;
  e = cudaFuncGetAttributes(&own, KERNEL);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)own.sharedSizeBytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}
// A launch as a dependent of the kernel before (paged.cuh: after_the_kernel_before), in clusters of `cluster` blocks
template <auto KERNEL, class Args> cudaError_t launch(dim3 grid, int threads, int smem, cudaStream_t s, const Args& P, int cluster = 1) {
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute at[2] = {};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension; at[1].val.clusterDim.x = (unsigned)cluster; at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  lc.gridDim = grid; lc.blockDim = dim3((unsigned)threads); lc.dynamicSmemBytes = (size_t)smem; lc.stream = s; lc.attrs = at; lc.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = smem > 48 * 1024 ? allow<KERNEL>() : cudaSuccess;
  return e == cudaSuccess ? cudaLaunchKernelEx(&lc, KERNEL, P) : e;
}

template <bool READ> int move(const ofa_kv_cache* c, const ofa_kv_batch* b, void* k, void* v, int n_rows, long long k_row, long long k_head, long long v_row,
                              long long v_head, void* stream) {
  paged::MoveArgs P;
  if (int rc = check_cache(c, b, n_rows, P.b, P.c)) return rc;
  if (n_rows == 0 || b->n_seqs == 0) return OFA_OK;
  const bool e4m3 = c->dtype == OFA_KV_E4M3;
  if (int rc = check_rows("k", k, {k_row, n_rows}, {k_head, c->n_kv_heads}, c->head_dim, READ)) return rc;
  if (int rc = check_rows("v", v, {v_row, n_rows}, {v_head, c->n_kv_heads}, c->head_dim, READ)) return rc;
  if (!READ && (overlap({c->page_stride, c->n_pages}, {c->head_stride, c->n_kv_heads}, {c->row_stride, c->page_size}, c->head_dim) ||
                (e4m3 && overlap({c->scale_page_stride, c->n_pages}, {c->scale_head_stride, c->n_kv_heads}, {c->scale_row_stride, c->page_size}, 1))))
    return fail(OFA_BAD_ARGUMENT, "rows of the cache overlap");
  if (READ ? k_row == v_row && k_head == v_head && twins({k_row, n_rows}, {k_head, c->n_kv_heads}, {0, 1}, c->head_dim, k, v, 2)
           : c->n_pages > 0 && (twins({c->page_stride, c->n_pages}, {c->head_stride, c->n_kv_heads}, {c->row_stride, c->page_size}, c->head_dim, c->k, c->v, e4m3 ? 1 : 2) ||
                                (e4m3 && twins({c->scale_page_stride, c->n_pages}, {c->scale_head_stride, c->n_kv_heads}, {c->scale_row_stride, c->page_size}, 1, c->k_scale, c->v_scale, 1))))
    return fail(OFA_BAD_ARGUMENT, "keys and values overlap where they are written");
  P.k = static_cast<bf16*>(k); P.v = static_cast<bf16*>(v); P.k_row = k_row; P.k_head = k_head; P.v_row = v_row; P.v_head = v_head;
  P.n_kv_heads = c->n_kv_heads; P.pair.set(2u * (unsigned)c->n_kv_heads);
  // four pieces of 16 bytes for a thread, in two turns, where there are rows for it: a block then amortises the search for its sequences
  const long long per_row = 2ll * c->n_kv_heads * (c->head_dim / (e4m3 ? 16 : 8));
  long long rows = (1024 + per_row - 1) / per_row;
  while (rows > 1 && (n_rows + rows - 1) / rows < 148) rows--;
  P.rows = (int)(rows < paged::MOVE_ROWS ? rows : paged::MOVE_ROWS);
  const unsigned grid = (unsigned)((n_rows + P.rows - 1) / P.rows);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool small = c->head_dim == 64;
  const cudaError_t e = e4m3 ? small ? launch<paged::move_kernel<64, true, READ>>(grid, 256, 0, s, P) : launch<paged::move_kernel<128, true, READ>>(grid, 256, 0, s, P)
                             : small ? launch<paged::move_kernel<64, false, READ>>(grid, 256, 0, s, P) : launch<paged::move_kernel<128, false, READ>>(grid, 256, 0, s, P);
  return launched(e, READ ? "ofa_kv_read" : "ofa_kv_append");
}

// ---- attention
struct Plan { bool many, cluster, by_head, ranked; int pair, rows, tiles, nsplit; size_t bytes; };      // rows: of a tile

// A chunk of more than 16 rows for a key/value head goes to the tensor-core kernel, which reads the keys once for 128 or 256 rows; fewer to the one that keeps more bytes
// in flight. max_new and max_kv are what the caller says; without them one sequence with all rows and the page table's width are assumed.
//
// How many blocks share a tile's keys: the number for which the call should take least, in units of 128 keys of a block: one block's time where all run at once, else all blocks' time over
// the places for them and half a block's more for the end. What a block costs beside its keys (its first loads one after the other, the meeting at its end) measured 3 units of the tensor-core
// kernel and 6 of the other, a second launch to join parts 3, and parts pass through memory at 5 TB/s, a unit being 1.6 us. Up to eight blocks of the few-row kernel are a cluster and need no parts.
// (64 tokens over 4,096 8-bit keys: 112 us with one block a tile, 108 with two, 121 with four; a token over 1,000 keys, 12 heads of 64: 10.3, 8.5, 6.8 and 6.2 us with one, two, four and
// eight; two over 131,072 keys: 176 with twelve, 158 with 16, 170 with 24, 200 with 32; five tokens of 64 sequences over 4,096 keys 176 and 224. It takes the second, the last, 24 and the first
// of these. Contexts are all taken for the longest: 64 uneven ones of up to 4,096 8-bit keys, the longest first, take 62 with one and 75 with two, which it chooses.)
Plan plan(const ofa_kv_cache* c, const ofa_kv_batch* b, int n_rows, int n_heads) {
  Plan p;
  const long long group = n_heads / c->n_kv_heads;
  const long long rows = (b->max_new > 0 && b->max_new < n_rows ? b->max_new : n_rows) * group;
  p.many = rows > 16;
  // Tiles a block of the tensor-core kernel. One where bf16 tiles are small, or where the rows are few: two blocks an SM then cover each other's waits (12 tokens of 24 sequences over
  // 2,000 keys: 50 us with one, 69 with two). 8-bit rows need the room for their own ring, one block an SM has twice the workers (83 -> 78; for heads of 64 no gain).
  p.pair = c->head_dim == 64 ? (c->dtype == OFA_KV_BF16 ? 1 : 2) : rows <= 64 ? 1 : 2;
  p.rows = p.many ? (p.pair == 1 && c->head_dim == 128 ? 64 : 128 * p.pair) : rows > 8 ? 16 : 8;
  long long tiles = (rows + p.rows - 1) / p.rows;
  if (tiles > 4096) tiles = 4096;
  if (tiles < 1) tiles = 1;
  const long long cap = (long long)b->max_pages * c->page_size, kv = b->max_kv > 0 && b->max_kv < cap ? b->max_kv : cap;
  const long long blocks = (long long)(b->n_seqs > 0 ? b->n_seqs : 1) * c->n_kv_heads * tiles, units = (kv + 127) / 128;
  const long long fewer = p.many ? std::min(rows / group, kv) / 256 : 0;       // units that a chunk's blocks have less on average than the last one
  const long long slots = 148 * (p.many ? (c->dtype == OFA_KV_BF16 ? 2 / p.pair : 1) : p.rows == 8 ? 3 : 2), fixed = p.many ? 3 : 6;
  const size_t part = (size_t)n_rows * n_heads * (c->head_dim + 2) * 4;      // bytes of one split's parts
  p.nsplit = 1;
  double best = 0;
  for (int ns : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
    const bool cluster = !p.many && ns <= 8;
    if (ns > 1 && (ns > units || (cluster && (ns & (ns - 1))) || blocks * ns > 0x7fffffffll)) continue;
    const double block = fixed + (double)((units + ns - 1) / ns), mean = fixed + (double)(units - fewer) / ns;
    const double t = (blocks * ns <= slots ? block : blocks * ns * mean / slots + block / 2) + (ns > 1 && !cluster ? 3 + 2.0 * part * ns / 8e6 : 0.0);
    if (ns == 1 || t < best) { best = t; p.nsplit = ns; p.cluster = cluster && ns > 1; }
  }
  // Keys and values of all heads above 48 MB are taken head by head (4,096 tokens over 16,384 keys of 8 heads, 67 MB: 850 us, 897 with all heads side by side); below that the longest
  // tiles of all heads go first (prompts of 1,024 tokens, 12.6 MB: 22.8 us, 29.4 head by head).
  p.by_head = (double)b->n_seqs * c->n_kv_heads * kv * c->head_dim * (c->dtype == OFA_KV_E4M3 ? 2 : 4) > 48e6;
  // Where blocks start one after the other, those of the longest sequences do so first (64 sequences over 1 to 4,096 keys: a token, 8-bit keys 76 us in the order of the table,
  // 67 so; five tokens 117 and 104, 8-bit keys 170 and 146). Every block ranks the lengths itself, 0.3 us.
  p.ranked = b->n_seqs > 1 && b->n_seqs <= 128 && blocks * p.nsplit > slots;
  p.tiles = (int)tiles;
  p.bytes = p.nsplit > 1 && !p.cluster ? part * p.nsplit : 0;
  return p;
}

// The pages as boxes of `run` rows for the copy engine; false where the driver will not have them, which leaves the other way of fetching them
bool map_pages(CUtensorMap* m, const void* base, const ofa_kv_cache* c, const paged::Pool& C, int run) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess ? (Encode)f : (Encode) nullptr;
  }();
  const bool e4m3 = c->dtype == OFA_KV_E4M3;
  const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size, (cuuint64_t)c->n_kv_heads, (cuuint64_t)c->n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)C.row_b, (cuuint64_t)C.head_b, (cuuint64_t)C.page_b};
  const cuuint32_t box[4] = {(cuuint32_t)(e4m3 ? c->head_dim : 64), (cuuint32_t)run, 1, 1}, one[4] = {1, 1, 1, 1};
  return encode && encode(m, e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          e4m3 && c->head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <int D, bool E4M3> cudaError_t attend(paged::AttnArgs& P, const Plan& p, cudaStream_t s) {
  const unsigned blocks = (unsigned)((long long)P.b.n_seqs * P.tiles * P.nsplit);
  cudaError_t e = cudaSuccess;
  if (p.many) {
    const dim3 grid(blocks * (unsigned)P.n_kv_heads);           // heads among the tiles, for the order in which blocks start
    P.flip = P.scale_log2 < 0.f;
    P.scale_log2 = fmaxf(fabsf(P.scale_log2), 1.17549435e-38f);      // the smallest normal number instead of 0: -inf times it has to stay -inf
    if constexpr (!E4M3 || D == 128) if (p.pair == 1) e = launch<paged::many_rows_kernel<D, E4M3, 1>>(grid, paged::Tc<D, E4M3, 1>::THREADS, paged::Tc<D, E4M3, 1>::SMEM, s, P);
    if constexpr (E4M3 || D == 128) if (p.pair == 2) e = launch<paged::many_rows_kernel<D, E4M3, 2>>(grid, paged::Tc<D, E4M3, 2>::THREADS, paged::Tc<D, E4M3, 2>::SMEM, s, P);
  } else {
    const dim3 grid(blocks * (unsigned)P.n_kv_heads);
    const int cluster = P.cluster ? P.nsplit : 1;
    e = p.rows == 8 ? launch<paged::few_rows_kernel<D, E4M3, 1>>(grid, 128, paged::Few<D, E4M3, 1>::SMEM, s, P, cluster)
                    : launch<paged::few_rows_kernel<D, E4M3, 2>>(grid, 128, paged::Few<D, E4M3, 2>::SMEM, s, P, cluster);
  }
  if (e == cudaSuccess && P.nsplit > 1 && !P.cluster) e = launch<paged::combine_kernel<D>>(dim3((unsigned)(((long long)P.b.n_rows * P.n_heads + 3) / 4)), 128, 0, s, P);
  return e;
}

// Where four vectors a thread still give every SM several blocks: the stream, and a block for each row's named tokens if they fit its table and the list of biases is short; else one kernel,
// with one vector a thread for few rows, since each block reads its row's whole history.
template <class T, bool WIDE> cudaError_t process(logits::Args& P, int rows, cudaStream_t s) {
  const int vn = Vec<T>::N, span = P.vocab + (WIDE ? vn - 1 : 0);
  const bool large = (long long)rows * ((span + 1024 * vn - 1) / (1024 * vn)) >= 4 * 148, words = P.tokens || P.bias_ids;
  const int stretch = (large ? 1024 : 256) * vn;
  const dim3 grid((unsigned)((span + stretch - 1) / stretch), (unsigned)rows);
  const long long named = (P.tokens ? P.max_tokens : 0) + (long long)P.max_bias;
  if (P.bias_ids && (!large || named > 8192 || P.max_bias > logits::SHORT_LIST))
    return large ? launch<logits::process_kernel<T, 4, WIDE, logits::SUMS>>(grid, 256, stretch * 8, s, P) : launch<logits::process_kernel<T, 1, WIDE, logits::SUMS>>(grid, 256, stretch * 8, s, P);
  if (!large || named > 8192) {
    const int smem = words ? stretch * 4 : 0;
    return large ? launch<logits::process_kernel<T, 4, WIDE, logits::WORDS>>(grid, 256, smem, s, P) : launch<logits::process_kernel<T, 1, WIDE, logits::WORDS>>(grid, 256, smem, s, P);
  }
  const cudaError_t e = launch<logits::process_kernel<T, 4, WIDE, logits::STREAM>>(grid, 256, 0, s, P);
  if (e != cudaSuccess || !words) return e;
  for (P.slots_log2 = 9; P.slots_log2 < 14 && 1ll << P.slots_log2 < 4 * named;) P.slots_log2++;
  return launch<logits::touch_kernel<T>>(dim3((unsigned)rows), 512, 12 << P.slots_log2, s, P);
}

}  // namespace

extern "C" const char* ofa_serving_last_error(void) { return g_error; }

extern "C" int ofa_kv_append(const ofa_kv_cache* cache, const ofa_kv_batch* batch, const void* k, const void* v, int n_rows, long long k_row_stride,
                             long long k_head_stride, long long v_row_stride, long long v_head_stride, void* stream) {
  return move<false>(cache, batch, const_cast<void*>(k), const_cast<void*>(v), n_rows, k_row_stride, k_head_stride, v_row_stride, v_head_stride, stream);
}
extern "C" int ofa_kv_read(const ofa_kv_cache* cache, const ofa_kv_batch* batch, void* k, void* v, int n_rows, long long k_row_stride, long long k_head_stride,
                           long long v_row_stride, long long v_head_stride, void* stream) {
  return move<true>(cache, batch, k, v, n_rows, k_row_stride, k_head_stride, v_row_stride, v_head_stride, stream);
}

extern "C" int ofa_paged_attention(const ofa_kv_cache* cache, const ofa_kv_batch* batch, const ofa_paged_attention_args* a, void* stream) {
  paged::AttnArgs P;
  if (!a) return fail(OFA_BAD_ARGUMENT, "null pointer");
  if (int rc = check_cache(cache, batch, a->n_rows, P.b, P.c)) return rc;
  if (a->n_heads < 1 || a->n_heads % cache->n_kv_heads) return fail(OFA_BAD_ARGUMENT, "n_heads %d is not a multiple of n_kv_heads %d", a->n_heads, cache->n_kv_heads);
  if (a->window < 0 || (a->window && !a->causal)) return fail(OFA_BAD_ARGUMENT, "window %d: a window (> 0) needs causal attention", a->window);
  if (!(a->scale > -1e30f && a->scale < 1e30f)) return fail(OFA_BAD_ARGUMENT, "scale is not finite");
  const long long group = a->n_heads / cache->n_kv_heads;
  if ((long long)a->n_rows * group > 0x7fffff00ll || (long long)a->n_rows * a->n_heads > 0x7fffff00ll * 4)
    return fail(OFA_BAD_ARGUMENT, "%d rows of %d heads are too many for one call", a->n_rows, a->n_heads);
  if (a->n_rows == 0 || batch->n_seqs == 0) return OFA_OK;
  if (int rc = check_rows("q", a->q, {a->q_row_stride, a->n_rows}, {a->q_head_stride, a->n_heads}, cache->head_dim, false)) return rc;
  if (int rc = check_rows("out", a->out, {a->out_row_stride, a->n_rows}, {a->out_head_stride, a->n_heads}, cache->head_dim, true)) return rc;
  if (!aligned(a->lse, 4)) return fail(OFA_BAD_ARGUMENT, "lse is misaligned");
  const Plan p = plan(cache, batch, a->n_rows, a->n_heads);
  if (p.bytes && (!a->workspace || a->workspace_bytes < p.bytes || !aligned(a->workspace, 16)))
    return fail(OFA_BAD_ARGUMENT, "workspace of %zu bytes on a 16-byte boundary needed, %zu given", p.bytes, a->workspace ? a->workspace_bytes : 0);
  if ((long long)batch->n_seqs * p.tiles * p.nsplit * cache->n_kv_heads > 0x7fffffffll) return fail(OFA_BAD_ARGUMENT, "%d sequences are too many for one call", batch->n_seqs);
  P.q = static_cast<const bf16*>(a->q); P.q_row = a->q_row_stride; P.q_head = a->q_head_stride;
  P.out = static_cast<bf16*>(a->out); P.o_row = a->out_row_stride; P.o_head = a->out_head_stride; P.lse = a->lse;
  P.n_heads = a->n_heads; P.n_kv_heads = cache->n_kv_heads; P.causal = a->causal != 0; P.window = a->window; P.group.set((unsigned)group);
  P.scale_log2 = a->scale * paged::LOG2E; P.flip = 0;
  P.wide = (long long)cache->n_pages * P.c.page_b + (long long)cache->page_size * P.c.row_b >= 1ll << 35; P.tiles = p.tiles; P.nsplit = p.nsplit; P.cluster = p.cluster; P.by_head = p.by_head; P.ranked = p.ranked; P.part = static_cast<float*>(a->workspace);
  // rows of a box of the copy engine: as many as divide a page and are of use at once, since a lane asks for one after the other
  P.run = std::min(cache->page_size & -cache->page_size, p.many ? 64 : cache->head_dim == 128 && cache->dtype == OFA_KV_BF16 ? 16 : 32);
  if (P.run < 8 || cache->n_pages == 0) P.run = 0;
  if (P.run && !(map_pages(&P.km, cache->k, cache, P.c, P.run) && map_pages(&P.vm, cache->v, cache, P.c, P.run))) P.run = 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (cache->dtype == OFA_KV_E4M3) e = cache->head_dim == 64 ? attend<64, true>(P, p, s) : attend<128, true>(P, p, s);
  else e = cache->head_dim == 64 ? attend<64, false>(P, p, s) : attend<128, false>(P, p, s);
  return launched(e, "ofa_paged_attention");
}

extern "C" size_t ofa_paged_attention_workspace(const ofa_kv_cache* cache, const ofa_kv_batch* batch, int n_rows, int n_heads) {
  paged::Batch B;
  paged::Pool C;
  if (check_cache(cache, batch, n_rows, B, C) || n_heads < 1 || n_heads % cache->n_kv_heads || n_rows == 0) return 0;
  return plan(cache, batch, n_rows, n_heads).bytes;
}

extern "C" int ofa_logits_process(const ofa_logits_args* a, void* stream) {
  if (!a) return fail(OFA_BAD_ARGUMENT, "null pointer");
  if (a->dtype != OFA_DTYPE_BF16 && a->dtype != OFA_DTYPE_F32) return fail(OFA_BAD_ARGUMENT, "logits dtype %d is neither OFA_DTYPE_BF16 nor OFA_DTYPE_F32", a->dtype);
  if (a->n_rows < 0 || a->vocab < 0 || a->max_tokens < 0 || a->max_bias < 0) return fail(OFA_BAD_ARGUMENT, "negative size: n_rows %d, vocab %d, max_tokens %d, max_bias %d", a->n_rows, a->vocab, a->max_tokens, a->max_bias);
  if (a->n_rows > 65535) return fail(OFA_BAD_ARGUMENT, "n_rows %d: at most 65535", a->n_rows);
  if (a->vocab > 1 << 30 || a->max_tokens > 1 << 29 || a->max_bias > 1 << 29)
    return fail(OFA_BAD_ARGUMENT, "vocab %d, max_tokens %d, max_bias %d: at most 2^30, 2^29 and 2^29", a->vocab, a->max_tokens, a->max_bias);
  if (a->n_rows == 0 || a->vocab == 0) return OFA_OK;
  const size_t es = a->dtype == OFA_DTYPE_F32 ? 4 : 2;
  if (!a->in || !a->out) return fail(OFA_BAD_ARGUMENT, "logits are null");
  if (!aligned(a->in, es) || !aligned(a->out, es)) return fail(OFA_BAD_ARGUMENT, "misaligned logits");
  if (a->out_stride < a->vocab && a->n_rows > 1) return fail(OFA_BAD_ARGUMENT, "rows of out overlap: stride %lld, vocab %d", a->out_stride, a->vocab);
  if (a->in_stride < 0 || a->tokens_stride < 0 || a->bias_stride < 0 || a->mask_stride < 0) return fail(OFA_BAD_ARGUMENT, "negative stride");
  {                                                              // in place, or apart: a row of out that lies on others of in would be read after it was written
    const intptr_t d = reinterpret_cast<intptr_t>(a->out) - reinterpret_cast<intptr_t>(a->in), row = (intptr_t)(a->vocab * es), st = (intptr_t)(a->out_stride * es);
    const intptr_t in_end = (intptr_t)((a->n_rows - 1) * a->in_stride * es) + row, out_end = (a->n_rows - 1) * st + row;
    const bool same = a->n_rows == 1 || a->in_stride == a->out_stride;
    const intptr_t off = st > 0 ? ((d % st) + st) % st : d;      // with equal strides: how far a row of out begins behind one of in
    const bool apart = d >= in_end || -d >= out_end || (a->n_rows > 1 && same && off >= row && st - off >= row);
    if (!apart && !(d == 0 && same)) return fail(OFA_BAD_ARGUMENT, "out and in overlap and are not the same");
  }
  if ((a->repetition || a->presence || a->frequency) && !a->tokens && a->max_tokens > 0) return fail(OFA_BAD_ARGUMENT, "penalties need tokens");
  if (!a->bias_ids != !a->bias) return fail(OFA_BAD_ARGUMENT, "bias_ids and bias come together");
  if (!aligned(a->tokens, 4) || !aligned(a->n_tokens, 4) || !aligned(a->n_prompt, 4) || !aligned(a->repetition, 4) || !aligned(a->presence, 4) || !aligned(a->frequency, 4) ||
      !aligned(a->bias_ids, 4) || !aligned(a->bias, 4) || !aligned(a->mask, 4)) return fail(OFA_BAD_ARGUMENT, "misaligned array");
  logits::Args P;
  P.in = a->in; P.out = a->out; P.in_row = a->in_stride; P.out_row = a->out_stride; P.vocab = a->vocab;
  const bool history = a->tokens && a->max_tokens > 0 && (a->repetition || a->presence || a->frequency);
  P.tokens = history ? a->tokens : nullptr; P.tokens_row = a->tokens_stride; P.max_tokens = a->max_tokens; P.n_tokens = a->n_tokens; P.n_prompt = a->n_prompt;
  P.repetition = a->repetition; P.presence = a->presence; P.frequency = a->frequency;
  P.bias_ids = a->max_bias > 0 ? a->bias_ids : nullptr; P.bias = a->bias; P.bias_row = a->bias_stride; P.max_bias = a->bias_ids ? a->max_bias : 0;
  P.mask = a->mask; P.mask_row = a->mask_stride;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // whole 16-byte vectors where rows of in and out lie alike against their boundaries (an odd vocabulary moves both from row to row)
  const bool wide = (reinterpret_cast<uintptr_t>(a->in) - reinterpret_cast<uintptr_t>(a->out)) % 16 == 0 && (a->n_rows == 1 || ((a->in_stride - a->out_stride) * (long long)es) % 16 == 0);
  const cudaError_t e = a->dtype == OFA_DTYPE_F32 ? wide ? process<float, true>(P, a->n_rows, s) : process<float, false>(P, a->n_rows, s)
                                                  : wide ? process<bf16, true>(P, a->n_rows, s) : process<bf16, false>(P, a->n_rows, s);
  return launched(e, "ofa_logits_process");
}
