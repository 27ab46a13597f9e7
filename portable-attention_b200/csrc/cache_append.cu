// pa_cache_append: write new tokens into a block-scaled cache.
//
// For a block of scale_block rows of one (sequence, kv head), with x its new
// rows and c, s the codes and scale of rows it holds already:
//   need = 2^ceil(log2(max|x| / qmax)),  s' = max(need, s),
//   new codes rne(x / s'),  old codes rne(c * s / s') where s' > s.
// Bytes: each new element is read once (2 bytes) and written once (1 byte); the
// arithmetic is a few operations per element, so the call is bound by memory,
// or by latency for a single token per sequence.
//
// One warp owns one (sequence, block, kv head, K or V), so a scale has one
// writer and its rows need no other synchronisation. Lanes take 16-byte pieces
// (8 elements) of consecutive rows. Up to eight pieces a lane (16 rows of 128, 32
// of 64) stay in registers between the maximum and the coding, so the input is
// read once; larger blocks are read again. Magnitudes compare as integers two at
// a time, and where s' is a power of two in fp16's range the coding is packed
// fp16 arithmetic that rounds once. The new rows are asked for before the page is
// known. 8 x 4096 tokens of 8 x 128 fp16 to e4m3 in 16-row blocks: 41.3 us, 4.9
// TB/s of the 204 MB that must move (75 % of the measured copy rate), with 24 warps
// an SM; bound by the chain length -> rows and page -> codes at that occupancy
// (issue slots half used). To fp16: 47.3 us for 268 MB (5.7 TB/s). Larger blocks have
// fewer warps and read their rows again: 128 rows 65 us, 1024 120, 4096 416. One token
// in each of 64 sequences: 6.3 us, the host call.
#include <math.h>

#include <cmath>
#include <string>

#include "cache.cuh"

namespace pa {

pa_status check_cache(const pa_block_cache_desc* d, const CacheUse& use, CacheView* v,
                      const char* who) {
  const std::string w = std::string(who) + ": ";
  if (!d) return fail(PA_ERR_INVALID, w + "null descriptor");
  const pa_kv_cache_desc& c = d->cache;
  constexpr int64_t kMax = 0x7fffffffLL;
  if (c.q_dtype != PA_F16 && c.q_dtype != PA_BF16) return fail(PA_ERR_UNSUPPORTED, w + "q dtype must be fp16 or bf16");
  if (c.kv_dtype != c.q_dtype && c.kv_dtype != PA_FP8_E4M3 && c.kv_dtype != PA_I8)
    return fail(PA_ERR_UNSUPPORTED, w + "the cache dtype must be the query's dtype, fp8 e4m3 or int8");
  if (c.head_dim != 64 && c.head_dim != 128) return fail(PA_ERR_UNSUPPORTED, w + "head dim must be 64 or 128");
  if (c.batch < 0 || c.batch > 65535 * 1024LL) return fail(PA_ERR_INVALID, w + "batch out of range");
  if (c.kv_heads < 1 || c.kv_heads > 65535) return fail(PA_ERR_INVALID, w + "kv_heads out of range");
  if (use.decode) {
    if (c.q_heads < 1 || c.q_heads % c.kv_heads) return fail(PA_ERR_INVALID, w + "q heads must be a multiple of kv heads");
    if (c.q_heads / c.kv_heads > 16) return fail(PA_ERR_UNSUPPORTED, w + "at most 16 query heads per key/value head");
    if (!std::isfinite(c.scale)) return fail(PA_ERR_INVALID, w + "scale must be finite");
  }
  if (c.k_scale != 1.f || c.v_scale != 1.f)
    return fail(PA_ERR_INVALID, w + "k_scale and v_scale must be 1 (the scales are per block)");
  if (c.max_seq_len < 0 || c.max_seq_len > kMax - 65536) return fail(PA_ERR_UNSUPPORTED, w + "too many keys");
  if (c.page_size < 1 || c.page_size > kMax) return fail(PA_ERR_INVALID, w + "page_size must be in [1, 2^31)");
  if (c.num_pages < 1 || c.num_pages > kMax) return fail(PA_ERR_INVALID, w + "num_pages must be in [1, 2^31)");
  const int esz = c.kv_dtype == PA_FP8_E4M3 || c.kv_dtype == PA_I8 ? 1 : 2;
  constexpr int64_t kMaxStride = 1LL << 46;
  if (c.key_stride < c.head_dim || c.head_stride < c.head_dim || c.page_stride < c.head_dim)
    return fail(PA_ERR_INVALID, w + "cache strides must be at least head_dim");
  if (c.key_stride > kMaxStride || c.head_stride > kMaxStride || c.page_stride > kMaxStride)
    return fail(PA_ERR_INVALID, w + "cache strides out of range");
  if (c.key_stride * esz % 16 || c.head_stride * esz % 16 || c.page_stride * esz % 16)
    return fail(PA_ERR_INVALID, w + "cache strides must be multiples of 16 bytes");
  if (use.paged) {
    if (c.max_pages_per_seq < 0 || c.max_pages_per_seq > kMax) return fail(PA_ERR_INVALID, w + "max_pages_per_seq out of range");
    if (c.max_pages_per_seq < (c.max_seq_len + c.page_size - 1) / c.page_size)
      return fail(PA_ERR_INVALID, w + "max_pages_per_seq * page_size must cover max_seq_len");
  } else {
    if (c.num_pages < c.batch) return fail(PA_ERR_INVALID, w + "without a block table the cache needs one page per sequence");
    if (c.page_size < c.max_seq_len) return fail(PA_ERR_INVALID, w + "without a block table page_size must be at least max_seq_len");
  }
  if (esz == 1) {
    if (d->scale_block < 1 || d->scale_block > kMax) return fail(PA_ERR_INVALID, w + "scale_block must be in [1, 2^31)");
    if (use.paged && c.page_size % d->scale_block) return fail(PA_ERR_INVALID, w + "scale_block must divide page_size");
    const int64_t blocks = (c.page_size + d->scale_block - 1) / d->scale_block;
    if (d->scale_head_stride < blocks || d->scale_page_stride < blocks)
      return fail(PA_ERR_INVALID, w + "scale strides must be at least the blocks of a page");
    if (d->scale_head_stride > kMaxStride || d->scale_page_stride > kMaxStride)
      return fail(PA_ERR_INVALID, w + "scale strides out of range");
  }
  if (use.rows) {
    if (d->row_head_stride < c.max_seq_len || d->row_seq_stride < c.max_seq_len)
      return fail(PA_ERR_INVALID, w + "row strides must be at least max_seq_len");
    if (d->row_head_stride > kMaxStride || d->row_seq_stride > kMaxStride)
      return fail(PA_ERR_INVALID, w + "row strides out of range");
  }
  *v = CacheView{};
  v->key_stride = c.key_stride * esz;
  v->head_stride = c.head_stride * esz;
  v->page_stride = c.page_stride * esz;
  v->scale_head = d->scale_head_stride;
  v->scale_page = d->scale_page_stride;
  v->row_head = d->row_head_stride;
  v->row_seq = d->row_seq_stride;
  v->B = static_cast<int32_t>(c.batch);
  v->Hq = use.decode ? static_cast<int32_t>(c.q_heads) : 0;
  v->Hkv = static_cast<int32_t>(c.kv_heads);
  v->D = static_cast<int32_t>(c.head_dim);
  v->page_size = static_cast<int32_t>(c.page_size);
  v->num_pages = static_cast<int32_t>(c.num_pages);
  v->max_pages = use.paged ? static_cast<int32_t>(c.max_pages_per_seq) : 1;
  // Blocks above a page (of a dense cache) are the page: no sum below passes 32 bits.
  v->scale_block = esz == 1 ? static_cast<int32_t>(d->scale_block < c.page_size ? d->scale_block : c.page_size) : 0;
  v->max_len = static_cast<int32_t>(c.max_seq_len);
  v->q_bf16 = c.q_dtype == PA_BF16;
  v->kind = c.kv_dtype == PA_FP8_E4M3 ? kCacheE4M3 : c.kv_dtype == PA_I8 ? kCacheI8 : v->q_bf16 ? kCacheBF16 : kCacheF16;
  v->paged = use.paged;
  v->by_page = make_fastdiv(static_cast<uint32_t>(v->page_size));
  v->by_block = make_fastdiv(static_cast<uint32_t>(v->scale_block > 0 ? v->scale_block : 1));
  return PA_OK;
}

pa_status check_cache_ptrs(const CacheView& v, const void* k, const void* vc, const void* ks,
                           const void* vs, const char* who) {
  const std::string w = std::string(who) + ": ";
  if (!k || !vc) return fail(PA_ERR_INVALID, w + "null cache pointer");
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(vc)) & 15)
    return fail(PA_ERR_INVALID, w + "cache pointers must be 16-byte aligned");
  if (cache_8bit(v.kind) && (!ks || !vs)) return fail(PA_ERR_INVALID, w + "8-bit caches need k_scales and v_scales");
  if (!cache_8bit(v.kind) && (ks || vs)) return fail(PA_ERR_INVALID, w + "16-bit caches have no scales");
  return PA_OK;
}

namespace {

struct AppendArgs {
  CacheView c;
  const uint8_t* x[2];  // new keys, new values
  uint8_t* cache[2];
  float* scales[2];
  const int32_t* table;
  const int32_t* lens;
  const int32_t* new_lens;
  const int32_t* start;
  float* weights;
  int32_t* positions;
  int32_t* lens_out;
  int* status;
  int64_t x_seq, x_tok, x_head;  // bytes
  int32_t T, blocks, rows_per_block;
  int64_t items;
};

// Eight 16-bit elements as codes of scale s. EASY: s is a power of two whose
// reciprocal fp16 holds as a normal number, and every element is finite.
template <int KIND, bool QBF16, bool EASY>
__device__ __forceinline__ uint2 encode8(const uint4& q, float s, float inv) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (EASY && !QBF16 && KIND == kCacheE4M3) {
    const __half r = __float2half_rn(inv);
    const __half2 r2 = __halves2half2(r, r);
    return make_uint2(e4m3_from_h4(h2_mul(w[0], r2), h2_mul(w[1], r2)),
                      e4m3_from_h4(h2_mul(w[2], r2), h2_mul(w[3], r2)));
  } else if constexpr (EASY && !QBF16) {
    const __half r = __float2half_rn(inv);
    const __half2 r2 = __halves2half2(r, r);
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // 1536 + x rounds to an integer whose low byte is the code
      const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&w[k]), r2, __floats2half2_rn(1536.f, 1536.f));
      o[k] = *reinterpret_cast<const uint32_t*>(&y);
    }
    return make_uint2(__byte_perm(o[0], o[1], 0x6420), __byte_perm(o[2], o[3], 0x6420));
  } else {
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = cache_unpack<QBF16>(w[k]);
      if (EASY && KIND == kCacheI8) {
        const float x = fmaf(f.x, inv, 12582912.f), y = fmaf(f.y, inv, 12582912.f);  // 1.5 * 2^23
        o[k] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x0040);
      } else if (EASY) {
        o[k] = cache_enc2<KIND>(f.x * inv, f.y * inv);
      } else {
        o[k] = cache_enc2<KIND>(__fdiv_rn(f.x, s), __fdiv_rn(f.y, s));
      }
    }
    return make_uint2(__byte_perm(o[0], o[1], 0x5410), __byte_perm(o[2], o[3], 0x5410));
  }
}

// kHold: pieces a lane holds, eight, or four for blocks that have no more (eight
// rows of 128: 65.7 us with eight, 55.5 with four, for 8 x 4096 tokens).
template <int KIND, int D, bool QBF16, int kHold>
__global__ void __launch_bounds__(256, kHold == 8 ? 3 : 4) cache_append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
  if (item >= a.items) return;
  // Heads vary fastest: token-major inputs and caches hold a token's heads side by side.
  const int h = static_cast<int>(item % a.c.Hkv);
  int64_t rest = item / a.c.Hkv;
  const int kv = static_cast<int>(rest & 1);
  rest >>= 1;
  const int blk = static_cast<int>(rest % a.blocks);
  const int b = static_cast<int>(rest / a.blocks);

  const int len = a.lens[b];
  int add = a.new_lens ? a.new_lens[b] : a.T;
  if (len < 0 || len > a.c.max_len || add < 0 || add > a.T || add > a.c.max_len - len) {
    if (lane == 0) atomicExch(a.status, kStatusBadSeqLen);
    add = 0;
  }
  if (a.lens_out && h == 0 && kv == 0 && blk == 0) {
    // A sequence some of whose new rows have no page keeps its length.
    bool wrong = false;
    if (a.table && add > 0) {
      const int32_t* pages = a.table + static_cast<int64_t>(b) * a.c.max_pages;
      const int last = fast_div(a.c.by_page, len + add - 1);
      for (int i = fast_div(a.c.by_page, len) + lane; i <= last; i += 32) {
        const int32_t page = pages[i];
        wrong = wrong || page < 0 || page >= a.c.num_pages;
      }
    }
    wrong = __any_sync(0xffffffffu, wrong);
    if (lane == 0) a.lens_out[b] = wrong ? len : len + add;
  }
  const int bs = a.rows_per_block;
  const int64_t r_first = (static_cast<int64_t>(len / bs) + blk) * bs;  // first row of this block
  if (add == 0 || r_first >= static_cast<int64_t>(len) + add) return;
  const int r0 = static_cast<int>(r_first);
  const int lo = r0 > len ? r0 : len;  // first new row
  const int hi = static_cast<int>(r_first + bs < static_cast<int64_t>(len) + add ? r_first + bs : len + add);

  constexpr int kChunks = D / 8;       // 16-byte pieces of a new row
  constexpr int kRows = 32 / kChunks;  // rows per step of the warp
  const int row_l = lane / kChunks, ch = lane % kChunks;
  // This lane's piece of row lo + row_l; its next is kRows rows on.
  const uint8_t* const src =
      (kv ? a.x[1] : a.x[0]) + b * a.x_seq + h * a.x_head + (lo - len + row_l) * a.x_tok + ch * 16;
  uint8_t* const cache = kv ? a.cache[1] : a.cache[0];
  const int rows = hi - lo;
  // Per-row arrays of the rows that have a page (in 8 bits all have the block's).
  auto set_rows = [&]() {
    if (kv != 0 || !(a.weights || a.positions)) return;
    const int64_t row0 = b * a.c.row_seq + h * a.c.row_head;
    const int p0 = a.positions ? (a.start ? a.start[b] : len) : 0;
    for (int r = lo + lane; r < hi; r += 32) {
      if (!cache_8bit(KIND) && cache_page(a.c, a.table, b, r, a.status) < 0) continue;
      if (a.weights) a.weights[row0 + r] = 0.f;
      if (a.positions) a.positions[row0 + r] = p0 + (r - len);
    }
  };

  uint4 x[kHold];
  const int64_t x_step = kRows * a.x_tok;
  auto read = [&](int first) {
    const uint8_t* p = src + first * a.x_tok;
    if (rows - first >= kHold * kRows) {
#pragma unroll
      for (int u = 0; u < kHold; ++u, p += x_step) x[u] = __ldcs(reinterpret_cast<const uint4*>(p));
      return;
    }
#pragma unroll
    for (int u = 0; u < kHold; ++u, p += x_step) {
      x[u] = make_uint4(0u, 0u, 0u, 0u);
      if (first + u * kRows + row_l < rows) x[u] = __ldcs(reinterpret_cast<const uint4*>(p));
    }
  };
  read(0);  // asked for before the page is known
  if (!cache_8bit(KIND)) {
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
      const int i = u * kRows + row_l;
      if (i >= rows) continue;
      const int32_t page = cache_page(a.c, a.table, b, lo + i, a.status);
      if (page < 0) continue;
      *reinterpret_cast<uint4*>(cache + cache_row(a.c, page, h, cache_at(a.c, lo + i)) + ch * 16) = x[u];
    }
    set_rows();
    return;
  }
  // 8 bits: the block lies in one page.
  const int32_t page = cache_page(a.c, a.table, b, lo, a.status);
  if (page < 0) return;
  set_rows();
  const int at0 = cache_at(a.c, r0);  // the block's first row inside its page
  float* const sp = (kv ? a.scales[1] : a.scales[0]) + cache_scale(a.c, page, h, at0);
  const bool held = r0 < len;  // earlier rows of this sequence live in the block
  const float old = held ? *sp : 0.f;
  // Largest magnitude, as 16-bit patterns; a pattern of `inf` or above is not finite.
  constexpr uint32_t kInf = QBF16 ? 0x7f80u : 0x7c00u;
  uint32_t top = 0u;
  for (int first = 0; first < rows; first += kHold * kRows) {
    if (first > 0) read(first);
#pragma unroll
    for (int u = 0; u < kHold; ++u)
      top = max_u16x2(max_u16x2(top, max_u16x2(x[u].x & 0x7fff7fffu, x[u].y & 0x7fff7fffu)),
                      max_u16x2(x[u].z & 0x7fff7fffu, x[u].w & 0x7fff7fffu));
  }
  top = __reduce_max_sync(0xffffffffu, (top & 0xffffu) > (top >> 16) ? top & 0xffffu : top >> 16);
  const bool finite = top < kInf;
  float amax = cache_unpack<QBF16>(top).x;
  if (!finite) {  // look again, passing over what is not
    amax = 0.f;
    for (int first = 0; first < rows; first += kHold * kRows) {
      if (rows > kHold * kRows) read(first);
#pragma unroll
      for (int u = 0; u < kHold; ++u) {
        const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = cache_unpack<QBF16>(w[k]);
          amax = cache_amax(cache_amax(amax, f.x), f.y);
        }
      }
    }
    amax = warp_max(amax);
  }
  const float need = cache_need_scale<KIND>(amax);
  const float s = old > need ? old : need;
  // 2^-15 <= s <= 2^14, a power of two: its reciprocal is a normal fp16 number.
  const bool easy = finite && cache_easy_ratio(1.f, s);
  const float inv = __fdiv_rn(1.f, s);
  uint8_t* const dst = cache + cache_row(a.c, page, h, at0) + ch * 8;
  uint8_t* const dst_l = dst + (lo - r0 + row_l) * a.c.key_stride;
  for (int first = 0; first < rows; first += kHold * kRows) {
    if (rows > kHold * kRows) read(first);
    if (easy) {
      uint8_t* p = dst_l + first * a.c.key_stride;
      const int64_t step = kRows * a.c.key_stride;
      if (rows - first >= kHold * kRows) {
#pragma unroll
        for (int u = 0; u < kHold; ++u, p += step) *reinterpret_cast<uint2*>(p) = encode8<KIND, QBF16, true>(x[u], s, inv);
      } else {
#pragma unroll
        for (int u = 0; u < kHold; ++u, p += step)
          if (first + u * kRows + row_l < rows) *reinterpret_cast<uint2*>(p) = encode8<KIND, QBF16, true>(x[u], s, inv);
      }
    } else {
#pragma unroll 1
      for (int u = 0; u < kHold; ++u) {
        const int i = first + u * kRows;
        if (i + row_l < rows) {
          const uint4 q = *reinterpret_cast<const uint4*>(src + i * a.x_tok);
          *reinterpret_cast<uint2*>(dst_l + i * a.c.key_stride) = encode8<KIND, QBF16, false>(q, s, inv);
        }
      }
    }
  }
  if (held && s != old) {
    // The scale grew: the block's earlier rows are coded again.
    const bool quick = cache_easy_ratio(old, s);
    const __half2 ratio = cache_ratio(old, s);
#pragma unroll 1
    for (int i = row_l; i < len - r0; i += kRows) {
      uint2* p = reinterpret_cast<uint2*>(dst + i * a.c.key_stride);
      const uint2 w = *p;
      if (quick) {
        *p = make_uint2(cache_rescale4<KIND>(w.x, ratio), cache_rescale4<KIND>(w.y, ratio));
        continue;
      }
      const uint32_t wd[2] = {w.x, w.y};
      uint32_t o[2] = {0u, 0u};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = cache_dec2<KIND>(wd[k >> 1] >> (16 * (k & 1)));
        o[k >> 1] |= cache_enc2<KIND>(__fdiv_rn(f.x * old, s), __fdiv_rn(f.y * old, s)) << (16 * (k & 1));
      }
      *p = make_uint2(o[0], o[1]);
    }
  }
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *sp = s;
}

template <int KIND, int D, bool QBF16>
pa_status launch_append(const AppendArgs& a, cudaStream_t st) {
  auto kern = a.rows_per_block <= 4 * 32 / (D / 8) ? cache_append_kernel<KIND, D, QBF16, 4> : cache_append_kernel<KIND, D, QBF16, 8>;
  const int64_t grid = (a.items + 7) / 8;
  kern<<<static_cast<unsigned>(grid), 256, 0, st>>>(a);
  PA_CUDA(cudaGetLastError());
  return PA_OK;
}

template <int D>
pa_status launch_append_kind(const AppendArgs& a, cudaStream_t st) {
  switch (a.c.kind) {
    case kCacheF16: return launch_append<kCacheF16, D, false>(a, st);
    case kCacheBF16: return launch_append<kCacheBF16, D, true>(a, st);
    case kCacheE4M3:
      return a.c.q_bf16 ? launch_append<kCacheE4M3, D, true>(a, st) : launch_append<kCacheE4M3, D, false>(a, st);
    default:
      return a.c.q_bf16 ? launch_append<kCacheI8, D, true>(a, st) : launch_append<kCacheI8, D, false>(a, st);
  }
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" pa_status pa_cache_append(const pa_block_cache_desc* desc, const void* k_new,
                                     const void* v_new, int64_t new_len, int64_t new_seq_stride,
                                     int64_t new_token_stride, int64_t new_head_stride,
                                     const int32_t* new_lens, void* k_cache, void* v_cache,
                                     float* k_scales, float* v_scales, const int32_t* block_table,
                                     const int32_t* seq_lens, float* weights, int32_t* positions,
                                     const int32_t* start_positions, int32_t* seq_lens_out,
                                     void* stream) {
  clear_error();
  AppendArgs a{};
  PA_TRY(check_cache(desc, {block_table != nullptr, weights || positions, false}, &a.c, "cache append"));
  // A padded batch may be wider than the cache: each sequence's count is checked on the device.
  if (new_len < 0 || new_len > (new_lens ? 0x7fffffffLL : a.c.max_len))
    return fail(PA_ERR_INVALID, "cache append: new_len must be in [0, max_seq_len], or below 2^31 with new_lens");
  if (start_positions && !positions) return fail(PA_ERR_INVALID, "cache append: start_positions without positions");
  if (a.c.B == 0) return PA_OK;
  if (!seq_lens) return fail(PA_ERR_INVALID, "cache append: null seq_lens");
  if (seq_lens_out == seq_lens) return fail(PA_ERR_INVALID, "cache append: seq_lens_out must not be seq_lens");
  if (seq_lens_out && (seq_lens_out == new_lens || seq_lens_out == start_positions))
    return fail(PA_ERR_INVALID, "cache append: seq_lens_out must not be new_lens or start_positions");
  if (new_len > 0) {
    PA_TRY(check_cache_ptrs(a.c, k_cache, v_cache, k_scales, v_scales, "cache append"));
    if (!k_new || !v_new) return fail(PA_ERR_INVALID, "cache append: null k_new or v_new");
    if ((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) & 15)
      return fail(PA_ERR_INVALID, "cache append: k_new and v_new must be 16-byte aligned");
    for (int64_t s : {new_seq_stride, new_token_stride, new_head_stride})
      if (s < 0 || s > (1LL << 46) || s % 8)
        return fail(PA_ERR_INVALID, "cache append: strides of the new tokens must be non-negative multiples of 8 elements");
  }
  a.x[0] = static_cast<const uint8_t*>(k_new);
  a.x[1] = static_cast<const uint8_t*>(v_new);
  a.cache[0] = static_cast<uint8_t*>(k_cache);
  a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.scales[0] = k_scales;
  a.scales[1] = v_scales;
  a.table = block_table;
  a.lens = seq_lens;
  a.new_lens = new_lens;
  a.start = start_positions;
  a.weights = weights;
  a.positions = positions;
  a.lens_out = seq_lens_out;
  a.x_seq = new_seq_stride * 2;
  a.x_tok = new_token_stride * 2;
  a.x_head = new_head_stride * 2;
  a.T = static_cast<int32_t>(new_len);
  // 16-bit caches have no blocks: 16 rows make an item (eight pieces a lane, or four).
  a.rows_per_block = cache_8bit(a.c.kind) ? a.c.scale_block : 16;
  // Blocks that the rows of a sequence, starting anywhere, can touch; one at least, for seq_lens_out.
  const int64_t bs = a.rows_per_block, most = a.T < a.c.max_len ? a.T : a.c.max_len;
  a.blocks = most > 0 ? static_cast<int32_t>((most + 2 * bs - 2) / bs) : 1;
  const int64_t per_block = static_cast<int64_t>(a.c.B) * 2 * a.c.Hkv;  // below 2^43
  if (a.blocks > 8 * 0x7fffffffLL / per_block) return fail(PA_ERR_UNSUPPORTED, "cache append: grid too large");
  a.items = per_block * a.blocks;
  a.status = device_status_word();
  if (!a.status) return fail(PA_ERR_CUDA, "device status word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a.c.D == 128 ? launch_append_kind<128>(a, st) : launch_append_kind<64>(a, st);
}
