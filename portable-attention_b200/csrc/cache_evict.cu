// pa_cache_evict: keep each (sequence, kv head)'s `budget` rows of the largest
// accumulated attention weight.
//
// Rows are ranked by an ordered 32-bit key: all ones for protected rows (the
// newest by position and the first ones), else the float's bits made monotonic,
// 0 for NaN. Kept are the n = budget largest, ties to the lowest row. Row r < n
// that is not kept is a hole; the k-th hole receives the k-th kept row at or
// above n. Sources lie at or above n and holes below, so no row is both read
// and written, every move is independent of the others, and only rows that must
// move are touched (an order-keeping compaction would move every row behind the
// first hole).
//
// Two launches. `select` finds the threshold key by radix selection (four
// passes of eight bits), the holes and their sources, and leaves in kept[] the
// row that each place gets. `move` carries the rows, their weights and
// positions over. In 8-bit caches a warp owns a whole scale block: it rescales
// the block by the rule of pa_cache_append. The block that `budget` cuts holds
// places below it and possibly sources at or above it; its old scale is put
// aside by `select`, since `move` changes it while other warps read from it.
#include <math.h>

#include "cache.cuh"

namespace pa {
namespace {

struct EvictArgs {
  CacheView c;
  uint8_t* cache[2];
  float* scales[2];
  const int32_t* table;
  const int32_t* lens;
  const float* weights;
  const int32_t* positions;
  const int32_t* next;
  float* weights_out;
  int32_t* positions_out;
  int32_t* lens_out;
  int32_t* kept;      // [B][Hkv][budget]
  int32_t* holes;     // workspace [B][Hkv][budget]
  float* cut_scale;   // workspace [B][Hkv][2]
  int* status;
  int32_t budget, recent, sinks;
  int32_t rows_per_block;
};

__device__ __forceinline__ int evict_len(const EvictArgs& a, int b, bool report) {
  const int n = a.lens[b];
  if (n >= 0 && n <= a.c.max_len) return n;
  if (report) atomicExch(a.status, kStatusBadSeqLen);
  return -1;
}

// Monotonic key of a weight; -0 counts as 0, NaN as the lowest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024;

// Inclusive ranks over the CTA of a flag; *total receives the CTA's count.
__device__ __forceinline__ int cta_rank(bool flag, int* warp_sum, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t m = __ballot_sync(0xffffffffu, flag);
  __syncthreads();  // earlier readers of warp_sum are done
  if (lane == 0) warp_sum[warp] = __popc(m);
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const int n = warp_sum[w];
    before += w < warp ? n : 0;
    all += n;
  }
  *total = all;
  return before + __popc(m & ((2u << lane) - 1u));
}

__global__ void __launch_bounds__(kSelThreads) cache_select_kernel(const EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int warp_sum[kSelThreads / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  const int h = blockIdx.x % a.c.Hkv, b = blockIdx.x / a.c.Hkv;
  const int tid = threadIdx.x;
  const int len = evict_len(a, b, tid == 0 && h == 0);
  const int n = a.budget;
  const int64_t pair = blockIdx.x;
  int32_t* kept = a.kept + pair * n;
  int32_t* holes = a.holes + pair * n;
  if (h == 0 && tid == 0) a.lens_out[b] = len < 0 ? a.lens[b] : (len < n ? len : n);
  if (len <= n) {
    for (int r = tid; r < n; r += kSelThreads) kept[r] = r < len ? r : -1;
    return;
  }
  if (cache_8bit(a.c.kind) && tid < 2 && n % a.rows_per_block) {
    // The cut block's scales, before `move` changes them.
    const int32_t page = cache_page(a.c, a.table, b, n, a.status);
    float s = 0.f;
    if (page >= 0) s = a.scales[tid][cache_scale(a.c, page, h, cache_at(a.c, n))];
    a.cut_scale[pair * 2 + tid] = s;
  }
  const float* w = a.weights + b * a.c.row_seq + h * a.c.row_head;
  const int32_t* pos = a.positions ? a.positions + b * a.c.row_seq + h * a.c.row_head : nullptr;
  const int64_t next = a.next ? a.next[b] : len;
  auto key_of = [&](int r) -> uint32_t {
    const int p = pos ? pos[r] : r;
    if (p >= next - a.recent || p < a.sinks) return 0xffffffffu;
    return weight_key(w[r]);
  };
  uint32_t prefix = 0;
  int left = n;  // rows still to take among those that match the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int r = tid; r < len; r += kSelThreads) {
      const uint32_t key = key_of(r);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255, t = left;
      while (d > 0 && hist[d] < t) t -= hist[d--];
      s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
      s_left = t;
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
  }
  // Rows above the key `prefix` are kept, and the first `left` rows that equal it.
  int ties = 0, n_holes = 0, n_src = 0;
  for (int base = 0; base < len; base += kSelThreads) {
    const int r = base + tid;
    const uint32_t key = r < len ? key_of(r) : 0u;
    const bool tie = r < len && key == prefix;
    int total;
    const int tie_rank = ties + cta_rank(tie, warp_sum, &total);
    ties += total;
    const bool keep = r < len && (key > prefix || (tie && tie_rank <= left));
    if (base < n) {
      const bool hole = r < n && !keep;
      const int rank = n_holes + cta_rank(hole, warp_sum, &total);
      n_holes += total;
      if (hole) holes[rank - 1] = r;
      if (r < n && keep) kept[r] = r;
      __syncthreads();  // the holes are in memory before a source looks one up
    }
    const bool src = r >= n && keep;
    const int rank = n_src + cta_rank(src, warp_sum, &total);
    n_src += total;
    if (src) kept[holes[rank - 1]] = r;
  }
}

// A warp moves the rows of one block of places of one (sequence, kv head).
template <int KIND, int D>
__global__ void __launch_bounds__(256) cache_move_kernel(const EvictArgs a, int32_t blocks, int64_t items) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
  if (item >= items) return;
  const int h = static_cast<int>(item % a.c.Hkv);
  const int64_t rest = item / a.c.Hkv;
  const int blk = static_cast<int>(rest % blocks);
  const int b = static_cast<int>(rest / blocks);
  const int len = evict_len(a, b, false);
  const int n = a.budget, bs = a.rows_per_block;
  const int64_t pair = static_cast<int64_t>(b) * a.c.Hkv + h;
  const int32_t* kept = a.kept + pair * n;
  const int lo = blk * bs;
  int hi = lo + bs < n ? lo + bs : n;
  hi = hi < len ? hi : len;
  if (lo >= hi) return;
  const int64_t row0 = b * a.c.row_seq + h * a.c.row_head;
  int moved = 0;
  for (int r = lo + lane; r < hi; r += 32) {
    const int src = kept[r];
    moved += src != r;
    if (a.weights_out) a.weights_out[row0 + r] = a.weights[row0 + src];
    if (a.positions_out) a.positions_out[row0 + r] = a.positions ? a.positions[row0 + src] : src;
  }
  moved = __reduce_add_sync(0xffffffffu, moved);
  if (moved == 0) return;
  const int32_t* table = a.table;
  constexpr int kPieces = D * cache_esz(KIND) / 16;  // 16-byte pieces of a row
  const int total = (hi - lo) * kPieces;
  auto place = [&](int r) { return cache_at(a.c, r); };

  if (!cache_8bit(KIND)) {
    for (int i = lane; i < total; i += 32) {
      const int r = lo + i / kPieces, ch = i % kPieces;
      const int src = kept[r];
      if (src == r) continue;
      const int32_t pd = cache_page(a.c, table, b, r, a.status), ps = cache_page(a.c, table, b, src, a.status);
      if (pd < 0 || ps < 0) continue;
      const int64_t d = cache_row(a.c, pd, h, place(r)) + ch * 16, s = cache_row(a.c, ps, h, place(src)) + ch * 16;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        *reinterpret_cast<uint4*>(a.cache[kv] + d) = *reinterpret_cast<const uint4*>(a.cache[kv] + s);
    }
    return;
  }
  const int32_t page = cache_page(a.c, table, b, lo, a.status);
  if (page < 0) return;
  const int cut = n % bs ? n / bs : -1;  // the block whose old scales were put aside
#pragma unroll 1
  for (int kv = 0; kv < 2; ++kv) {
    auto src_scale = [&](int32_t ps, int src) -> float {
      if (src / bs == cut) return a.cut_scale[pair * 2 + kv];
      return a.scales[kv][cache_scale(a.c, ps, h, place(src))];
    };
    float amax = 0.f;
    for (int i = lane; i < total; i += 32) {
      const int r = lo + i / kPieces, ch = i % kPieces;
      const int src = kept[r];
      if (src == r) continue;
      const int32_t ps = cache_page(a.c, table, b, src, a.status);
      if (ps < 0) continue;
      const float s = src_scale(ps, src);
      const uint4 w = *reinterpret_cast<const uint4*>(a.cache[kv] + cache_row(a.c, ps, h, place(src)) + ch * 16);
      const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 f = cache_dec2<KIND>(wd[k >> 1] >> (16 * (k & 1)));
        amax = cache_amax(cache_amax(amax, f.x * s), f.y * s);
      }
    }
    amax = warp_max(amax);
    float* sp = a.scales[kv] + cache_scale(a.c, page, h, place(lo));
    const bool held = moved < hi - lo;
    const float need = cache_need_scale<KIND>(amax);
    const float old = held ? *sp : 0.f;
    const float s_new = old > need ? old : need;
    for (int i = lane; i < total; i += 32) {
      const int r = lo + i / kPieces, ch = i % kPieces;
      const int src = kept[r];
      if (src == r && s_new == old) continue;
      const int32_t ps = src == r ? page : cache_page(a.c, table, b, src, a.status);
      if (ps < 0) continue;
      const float s = src == r ? old : src_scale(ps, src);
      const uint4 w = *reinterpret_cast<const uint4*>(a.cache[kv] + cache_row(a.c, ps, h, place(src)) + ch * 16);
      const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
      uint32_t o[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 f = cache_dec2<KIND>(wd[k >> 1] >> (16 * (k & 1)));
        o[k >> 1] |= cache_enc2<KIND>(__fdiv_rn(f.x * s, s_new), __fdiv_rn(f.y * s, s_new)) << (16 * (k & 1));
      }
      *reinterpret_cast<uint4*>(a.cache[kv] + cache_row(a.c, page, h, place(r)) + ch * 16) =
          make_uint4(o[0], o[1], o[2], o[3]);
    }
    __syncwarp();  // every lane has read the old scale
    if (lane == 0) *sp = s_new;
  }
}

struct EvictPlan {
  CacheView c;
  size_t bytes;
};

pa_status plan_evict(const pa_block_cache_desc* d, bool paged, int64_t budget, EvictPlan* p) {
  *p = EvictPlan{};
  PA_TRY(check_cache(d, {paged, true, false}, &p->c, "cache evict"));
  if (budget < 1 || budget > 0x7fffffffLL - 1024) return fail(PA_ERR_INVALID, "cache evict: budget must be in [1, 2^31)");
  const size_t pairs = static_cast<size_t>(p->c.B) * p->c.Hkv;
  p->bytes = pairs * (2 * sizeof(float) + static_cast<size_t>(budget) * sizeof(int32_t));
  if (pairs > 0x7fffffffu) return fail(PA_ERR_UNSUPPORTED, "cache evict: grid too large");
  return PA_OK;
}

template <int KIND, int D>
pa_status launch_evict(const EvictArgs& a, cudaStream_t st) {
  cache_select_kernel<<<static_cast<unsigned>(a.c.B) * a.c.Hkv, kSelThreads, 0, st>>>(a);
  PA_CUDA(cudaGetLastError());
  const int32_t top = a.budget < a.c.max_len ? a.budget : a.c.max_len;
  const int32_t blocks = static_cast<int32_t>((static_cast<int64_t>(top) + a.rows_per_block - 1) / a.rows_per_block);
  const int64_t items = static_cast<int64_t>(a.c.B) * a.c.Hkv * blocks;
  if (items == 0) return PA_OK;
  if ((items + 7) / 8 > 0x7fffffffLL) return fail(PA_ERR_UNSUPPORTED, "cache evict: grid too large");
  cache_move_kernel<KIND, D><<<static_cast<unsigned>((items + 7) / 8), 256, 0, st>>>(a, blocks, items);
  PA_CUDA(cudaGetLastError());
  return PA_OK;
}

template <int D>
pa_status launch_evict_kind(const EvictArgs& a, cudaStream_t st) {
  switch (a.c.kind) {
    case kCacheF16:
    case kCacheBF16: return launch_evict<kCacheF16, D>(a, st);  // rows are copied as bits
    case kCacheE4M3: return launch_evict<kCacheE4M3, D>(a, st);
    default: return launch_evict<kCacheI8, D>(a, st);
  }
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" pa_status pa_cache_evict_workspace_size(const pa_block_cache_desc* desc, int32_t paged,
                                                   int64_t budget, size_t* bytes) {
  clear_error();
  if (!bytes) return fail(PA_ERR_INVALID, "null argument");
  EvictPlan p;
  PA_TRY(plan_evict(desc, paged != 0, budget, &p));
  *bytes = p.bytes;
  return PA_OK;
}

extern "C" pa_status pa_cache_evict(const pa_block_cache_desc* desc, void* k_cache, void* v_cache,
                                    float* k_scales, float* v_scales, const int32_t* block_table,
                                    const int32_t* seq_lens, const float* weights,
                                    const int32_t* positions, const int32_t* next_positions,
                                    int64_t budget, int64_t recent, int64_t sinks,
                                    float* weights_out, int32_t* positions_out,
                                    int32_t* seq_lens_out, int32_t* kept, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  clear_error();
  EvictPlan p;
  PA_TRY(plan_evict(desc, block_table != nullptr, budget, &p));
  if (recent < 0 || sinks < 0 || recent > budget || sinks > budget - recent)
    return fail(PA_ERR_INVALID, "cache evict: recent and sinks must be non-negative and fit the budget together");
  if (positions && !next_positions) return fail(PA_ERR_INVALID, "cache evict: positions need next_positions");
  if (p.c.B == 0) return PA_OK;
  if (!seq_lens || !weights || !seq_lens_out || !kept)
    return fail(PA_ERR_INVALID, "cache evict: null seq_lens, weights, seq_lens_out or kept pointer");
  if (seq_lens_out == seq_lens) return fail(PA_ERR_INVALID, "cache evict: seq_lens_out must not be seq_lens");
  PA_TRY(check_cache_ptrs(p.c, k_cache, v_cache, k_scales, v_scales, "cache evict"));
  if (workspace && workspace_bytes < p.bytes)
    return fail(PA_ERR_INVALID, "cache evict: workspace smaller than pa_cache_evict_workspace_size");
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(PA_ERR_INVALID, "cache evict: workspace must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  EvictArgs a{};
  a.c = p.c;
  a.cache[0] = static_cast<uint8_t*>(k_cache);
  a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.scales[0] = k_scales;
  a.scales[1] = v_scales;
  a.table = block_table;
  a.lens = seq_lens;
  a.weights = weights;
  a.positions = positions;
  a.next = next_positions;
  a.weights_out = weights_out;
  a.positions_out = positions_out;
  a.lens_out = seq_lens_out;
  a.kept = kept;
  a.status = device_status_word();
  if (!a.status) return fail(PA_ERR_CUDA, "device status word unavailable");
  a.budget = static_cast<int32_t>(budget);
  a.recent = static_cast<int32_t>(recent);
  a.sinks = static_cast<int32_t>(sinks);
  // 16-bit caches have no blocks: 16 rows make an item.
  a.rows_per_block = cache_8bit(p.c.kind) ? p.c.scale_block : 16;
  void* own = nullptr;
  if (!workspace) PA_TRY(scratch_alloc(&own, p.bytes, st));
  a.cut_scale = static_cast<float*>(workspace ? workspace : own);
  a.holes = reinterpret_cast<int32_t*>(a.cut_scale + static_cast<size_t>(p.c.B) * p.c.Hkv * 2);
  pa_status rc = p.c.D == 128 ? launch_evict_kind<128>(a, st) : launch_evict_kind<64>(a, st);
  scratch_free(own, st);
  return rc;
}
