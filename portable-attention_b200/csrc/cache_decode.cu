// pa_cache_decode: one query row per sequence attends to a block-scaled cache.
//
// With codes k8, v8 and their blocks' scales ks, vs:
//   s_j = scale * ks_j * (q . k8_j),  p = softmax(s),  out = sum_j p_j vs_j v8_j,
// and weights[b][h][j] += sum over the group's query heads of p_j. Each cached
// row is read once for all G query heads of its kv head.
//
// Two launches: `partial` splits every (sequence, kv head)'s keys over CTAs and
// leaves each split's running max, sum and accumulator (and, with weights, every
// score) in the workspace; `finish` joins the splits by log-sum-exp, writes the
// output and adds the weights.
#include <math.h>

#include <type_traits>

#include "cache.cuh"

namespace pa {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kWarps = 8;

struct DecodeArgs {
  CacheView c;
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* table;
  const int32_t* lens;
  void* out;
  float* lse;
  float* weights;
  float* ws_acc;     // [B*Hq][nsplit][D]
  float* ws_ml;      // [B*Hq][nsplit][2]: running max (log2 units), sum
  float* ws_scores;  // [B*Hq][score_stride] in log2 units, with weights only
  int* status;
  int64_t score_stride;
  int32_t G, nsplit, chunk;
  float scale_log2;
};

__device__ __forceinline__ int seq_len(const DecodeArgs& a, int b, bool report) {
  if (!a.lens) return a.c.max_len;
  const int n = a.lens[b];
  if (n >= 0 && n <= a.c.max_len) return n;
  if (report) atomicExch(a.status, kStatusBadSeqLen);
  return n < 0 ? 0 : a.c.max_len;
}

// E consecutive elements of a cached row as floats.
template <int KIND, int E>
__device__ __forceinline__ void load_elems(const uint8_t* row, int lane, float (&x)[E]) {
  if (cache_8bit(KIND)) {
    uint32_t w;
    if (E == 4)
      w = *reinterpret_cast<const uint32_t*>(row + lane * 4);
    else
      w = *reinterpret_cast<const uint16_t*>(row + lane * 2);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 f = cache_dec2<KIND>(w >> (16 * i));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 f = cache_unpack<KIND == kCacheBF16>(reinterpret_cast<const uint32_t*>(row)[lane * (E / 2) + i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

template <int KIND, int D, bool QBF16, int GT>
__global__ void __launch_bounds__(32 * kWarps) cache_partial_kernel(const DecodeArgs a) {
  constexpr int E = D / 32;  // elements of a row per lane
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % a.nsplit;
  const int pair = blockIdx.x / a.nsplit;
  const int b = pair / a.c.Hkv, h = pair % a.c.Hkv;
  const int G = a.G;
  const int len = seq_len(a, b, threadIdx.x == 0 && split == 0 && h == 0);
  const int64_t first = static_cast<int64_t>(split) * a.chunk;
  const int k0 = static_cast<int>(first < len ? first : len);
  const int k1 = static_cast<int>(first + a.chunk < len ? first + a.chunk : len);
  const int64_t q0 = static_cast<int64_t>(b) * a.c.Hq + static_cast<int64_t>(h) * G;

  float q[GT][E], acc[GT][E], m[GT], l[GT];
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      acc[g][e] = 0.f;
      q[g][e] = 0.f;
      if (g < G) {
        const int64_t i = (q0 + g) * D + lane * E + e;
        q[g][e] = QBF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[i])
                        : __half2float(static_cast<const __half*>(a.q)[i]);
      }
    }
  }
  for (int r = k0 + warp; r < k1; r += kWarps) {
    const int32_t page = cache_page(a.c, a.table, b, r, a.status);
    const int at = a.table ? r % a.c.page_size : r;
    float x[E], y[E], kscale = 1.f, vscale = 1.f;
    if (page >= 0) {
      const int64_t off = cache_row(a.c, page, h, at);
      load_elems<KIND, E>(a.k + off, lane, x);
      load_elems<KIND, E>(a.v + off, lane, y);
      if (cache_8bit(KIND)) {
        const int64_t so = cache_scale(a.c, page, h, at);
        kscale = a.ks[so];
        vscale = a.vs[so];
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = y[e] = 0.f;
    }
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      if (g >= G) break;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[g][e], x[e], s);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s *= a.scale_log2 * kscale;
      if (a.weights && lane == 0) a.ws_scores[(q0 + g) * a.score_stride + r] = s;
      const float mn = fmaxf(m[g], s);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float alpha = ex2(m[g] - base), p = ex2(s - base);
      m[g] = mn;
      l[g] = l[g] * alpha + p;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] = fmaf(p * vscale, y[e], acc[g][e] * alpha);
    }
  }
  __shared__ float sm[kWarps][GT], sl[kWarps][GT], sa[kWarps][D];
#pragma unroll
  for (int g = 0; g < GT; ++g)
    if (lane == 0) {
      sm[warp][g] = m[g];
      sl[warp][g] = l[g];
    }
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    if (g >= G) break;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) sa[warp][lane * E + e] = acc[g][e];
    __syncthreads();
    const int d = threadIdx.x;
    if (d < D) {
      float M = -INFINITY;
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w][g]);
      const float base = M == -INFINITY ? 0.f : M;
      float o = 0.f, L = 0.f;
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(sm[w][g] - base);
        o = fmaf(f, sa[w][d], o);
        L = fmaf(f, sl[w][g], L);
      }
      const int64_t slot = (q0 + g) * a.nsplit + split;
      a.ws_acc[slot * D + d] = o;
      if (d == 0) {
        a.ws_ml[slot * 2] = M;
        a.ws_ml[slot * 2 + 1] = L;
      }
    }
  }
}

// grid.x = B * Hkv pairs, grid.y: 0 writes the outputs, y >= 1 the weights of
// rows [(y - 1) * kRowsPerCta, ...).
constexpr int kRowsPerCta = 2048;

template <int D, bool QBF16>
__global__ void __launch_bounds__(256) cache_finish_kernel(const DecodeArgs a) {
  const int pair = blockIdx.x;
  const int b = pair / a.c.Hkv, h = pair % a.c.Hkv;
  const int64_t q0 = static_cast<int64_t>(b) * a.c.Hq + static_cast<int64_t>(h) * a.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float lse2[16];
  // Each warp joins the sums of its heads.
  for (int g = warp; g < a.G; g += 8) {
    const float* ml = a.ws_ml + (q0 + g) * a.nsplit * 2;
    float M = -INFINITY, L = 0.f;
    for (int s = lane; s < a.nsplit; s += 32) M = fmaxf(M, ml[2 * s]);
    M = warp_max(M);
    const float base = M == -INFINITY ? 0.f : M;
    for (int s = lane; s < a.nsplit; s += 32) L = fmaf(ex2(ml[2 * s] - base), ml[2 * s + 1], L);
#pragma unroll
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) lse2[g] = L > 0.f ? M + log2f(L) : (L == 0.f ? -INFINITY : L);
  }
  __syncthreads();
  if (blockIdx.y == 0) {
    for (int i = threadIdx.x; i < a.G * D; i += 256) {
      const int g = i / D, d = i % D;
      const float* ml = a.ws_ml + (q0 + g) * a.nsplit * 2;
      const float* acc = a.ws_acc + (q0 + g) * a.nsplit * D + d;
      const float z = lse2[g];
      float o = 0.f;
      if (z != -INFINITY)
        for (int s = 0; s < a.nsplit; ++s) {
          const float ms = ml[2 * s];
          if (ms != -INFINITY) o = fmaf(ex2(ms - z), acc[static_cast<int64_t>(s) * D], o);
        }
      if (QBF16)
        static_cast<__nv_bfloat16*>(a.out)[(q0 + g) * D + d] = __float2bfloat16_rn(o);
      else
        static_cast<__half*>(a.out)[(q0 + g) * D + d] = __float2half_rn(o);
      if (a.lse && d == 0) a.lse[q0 + g] = z * kLn2;
    }
    return;
  }
  const int len = seq_len(a, b, false);
  const int64_t r0 = static_cast<int64_t>(blockIdx.y - 1) * kRowsPerCta;
  const int r1 = static_cast<int>(r0 + kRowsPerCta < len ? r0 + kRowsPerCta : len);
  float* w = a.weights + b * a.c.row_seq + h * a.c.row_head;
  for (int64_t r = r0 + threadIdx.x; r < r1; r += 256) {
    float p = 0.f;
    for (int g = 0; g < a.G; ++g)
      if (lse2[g] != -INFINITY) p += ex2(a.ws_scores[(q0 + g) * a.score_stride + r] - lse2[g]);
    w[r] += p;
  }
}

struct DecodePlan {
  CacheView c;
  int G, nsplit, chunk;
  int64_t score_stride;
  bool weights;
  size_t bytes;
};

// Splits of a (sequence, kv head): enough CTAs for four waves, at least 64 keys each.
pa_status plan_decode(const pa_block_cache_desc* d, bool paged, bool weights, DecodePlan* p) {
  *p = DecodePlan{};
  PA_TRY(check_cache(d, {paged, weights, true}, &p->c, "cache decode"));
  p->G = p->c.Hq / p->c.Hkv;
  p->weights = weights;
  const int64_t pairs = static_cast<int64_t>(p->c.B) * p->c.Hkv;
  int64_t ns = pairs ? (4 * static_cast<int64_t>(sm_count()) + pairs - 1) / pairs : 1;
  const int64_t most = (p->c.max_len + 63) / 64;
  ns = ns > most ? most : ns;
  ns = ns > 256 ? 256 : ns < 1 ? 1 : ns;
  const int64_t chunk = (p->c.max_len + ns - 1) / ns;
  p->chunk = static_cast<int>(chunk < 1 ? 1 : chunk);
  p->nsplit = static_cast<int>(ns);
  p->score_stride = (static_cast<int64_t>(p->c.max_len) + 3) / 4 * 4;
  const size_t heads = static_cast<size_t>(p->c.B) * p->c.Hq;
  p->bytes = heads * p->nsplit * (p->c.D + 2) * sizeof(float);
  if (weights) p->bytes += heads * p->score_stride * sizeof(float);
  if (pairs * p->nsplit > 0x7fffffffLL) return fail(PA_ERR_UNSUPPORTED, "cache decode: grid too large");
  return PA_OK;
}

template <int KIND, int D, bool QBF16>
pa_status launch_decode(const DecodePlan& p, const DecodeArgs& a, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(p.c.B) * p.c.Hkv * p.nsplit;
  if (p.G <= 4)
    cache_partial_kernel<KIND, D, QBF16, 4><<<grid, 32 * kWarps, 0, st>>>(a);
  else
    cache_partial_kernel<KIND, D, QBF16, 16><<<grid, 32 * kWarps, 0, st>>>(a);
  PA_CUDA(cudaGetLastError());
  const unsigned y = p.weights ? 1 + (p.c.max_len + kRowsPerCta - 1) / kRowsPerCta : 1;
  if (y > 65535) return fail(PA_ERR_UNSUPPORTED, "cache decode: too many keys for weights");
  cache_finish_kernel<D, QBF16><<<dim3(static_cast<unsigned>(p.c.B) * p.c.Hkv, y), 256, 0, st>>>(a);
  PA_CUDA(cudaGetLastError());
  return PA_OK;
}

template <int D>
pa_status launch_decode_kind(const DecodePlan& p, const DecodeArgs& a, cudaStream_t st) {
  switch (p.c.kind) {
    case kCacheF16: return launch_decode<kCacheF16, D, false>(p, a, st);
    case kCacheBF16: return launch_decode<kCacheBF16, D, true>(p, a, st);
    case kCacheE4M3:
      return p.c.q_bf16 ? launch_decode<kCacheE4M3, D, true>(p, a, st) : launch_decode<kCacheE4M3, D, false>(p, a, st);
    default:
      return p.c.q_bf16 ? launch_decode<kCacheI8, D, true>(p, a, st) : launch_decode<kCacheI8, D, false>(p, a, st);
  }
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" pa_status pa_cache_decode_workspace_size(const pa_block_cache_desc* desc, int32_t paged,
                                                    int32_t with_weights, size_t* bytes) {
  clear_error();
  if (!bytes) return fail(PA_ERR_INVALID, "null argument");
  DecodePlan p;
  PA_TRY(plan_decode(desc, paged != 0, with_weights != 0, &p));
  *bytes = p.bytes;
  return PA_OK;
}

extern "C" pa_status pa_cache_decode(const pa_block_cache_desc* desc, const void* q,
                                     const void* k_cache, const void* v_cache,
                                     const float* k_scales, const float* v_scales,
                                     const int32_t* block_table, const int32_t* seq_lens, void* out,
                                     float* lse, float* weights, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  clear_error();
  DecodePlan p;
  PA_TRY(plan_decode(desc, block_table != nullptr, weights != nullptr, &p));
  if (p.c.B == 0) return PA_OK;
  if (!q || !out) return fail(PA_ERR_INVALID, "cache decode: null q or out pointer");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
    return fail(PA_ERR_INVALID, "cache decode: q and out must be 16-byte aligned");
  PA_TRY(check_cache_ptrs(p.c, k_cache, v_cache, k_scales, v_scales, "cache decode"));
  if (workspace && workspace_bytes < p.bytes)
    return fail(PA_ERR_INVALID, "cache decode: workspace smaller than pa_cache_decode_workspace_size");
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(PA_ERR_INVALID, "cache decode: workspace must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  DecodeArgs a{};
  a.c = p.c;
  a.q = q;
  a.k = static_cast<const uint8_t*>(k_cache);
  a.v = static_cast<const uint8_t*>(v_cache);
  a.ks = k_scales;
  a.vs = v_scales;
  a.table = block_table;
  a.lens = seq_lens;
  a.out = out;
  a.lse = lse;
  a.weights = weights;
  a.status = device_status_word();
  if (!a.status) return fail(PA_ERR_CUDA, "device status word unavailable");
  a.score_stride = p.score_stride;
  a.G = p.G;
  a.nsplit = p.nsplit;
  a.chunk = p.chunk;
  a.scale_log2 = static_cast<float>(desc->cache.scale * 1.4426950408889634);
  void* own = nullptr;
  if (!workspace) PA_TRY(scratch_alloc(&own, p.bytes, st));
  const size_t slots = static_cast<size_t>(p.c.B) * p.c.Hq * p.nsplit;
  a.ws_acc = static_cast<float*>(workspace ? workspace : own);
  a.ws_ml = a.ws_acc + slots * p.c.D;
  a.ws_scores = a.ws_ml + slots * 2;
  pa_status rc = p.c.D == 128 ? launch_decode_kind<128>(p, a, st) : launch_decode_kind<64>(p, a, st);
  scratch_free(own, st);
  return rc;
}
