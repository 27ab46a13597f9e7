// pa_cache_decode: one query row per sequence attends to a block-scaled cache.
//
// With codes k8, v8 and their blocks' scales ks, vs:
//   s_j = scale * ks_j * (q . k8_j),  p = softmax(s),  out = sum_j p_j vs_j v8_j,
// and weights[b][h][j] += sum over the group's query heads of p_j. Each cached
// row is read once for all G query heads of its kv head, so the call is bound by
// the cache's bytes.
//
// Work unit: (sequence, kv head, split) -> one CTA of four warps, three CTAs per
// SM (two for groups above 8, whose fragments need the registers), so that one
// streams while another starts or merges. Warp w owns tiles w, w + 4, ... of the
// CTA's keys (a tile is 4 KB of keys and 4 KB of values: 16, 32 or 64 rows) and
// two (three) shared-memory stages that it fills by cp.async as soon as it has
// used them; warps meet only to merge. cp.async takes an address per row, so
// pages may have any size and a row that does not exist (behind the length, or on
// a bad page) is filled with zeros and never read. The scales of a tile's rows
// come with it.
//
// Per tile, on tensor cores (m16n8k16, fp32 accumulators), operand layout as in
// decode.cu: S = Q K^T with the G query heads as rows, then O^T = V^T P^T with P
// straight from the S accumulators, taken relative to the tile:
//   p'_j = 2^(s_j - m_tile) * vs_j / 2^e * 2^14,  2^e <= max|vs| < 2^(e+1)
// (2^15 where there are no scales), and the tile's O^T joins the running one in
// fp32 with the factor 2^(m_tile - m_run) * 2^(e-14). A power of two is exact at both
// ends of fp32's range, where a reciprocal of max|vs| is not.
//
// p' goes in as two 16-bit terms, its leading bits cut off and what they leave: 20
// bits in fp16 while p is above 2^-18 of its tile's largest, then an absolute 2^-39 of
// that, whatever the other tiles hold (a first token that takes nearly all the
// weight, as trained models have, costs the others nothing); 14 bits for bf16 caches,
// which need bf16 products. With up to four heads the second terms are columns 4 to
// 7 of P^T, which would be empty: rows 4 to 7 of Q repeat the heads, the sums of both
// columns meet in the merge, and little is paid (64 x 8 x 32768 e4m3: 632 us with one
// term, 638 with two; the same time in fp16). Larger groups take products of their
// own (16 x 8 x 32768 e4m3: 8 heads 183 and 196 us, 16 heads 235 and 274; 32 x 8 x
// 4097 fp16 the same time). One term of 11 bits puts 1e-4 to 3e-4 of the output
// between this kernel and fp32 arithmetic, two less than 7e-5, all of it the
// rounding of the output.
//
// In bf16 caches p' has the factor 2^-5: bf16 has the range, and a tile's 32 rows near
// its end must not overflow. The running O^T carries a factor 2^-k, 2^k >= max_len:
// sums over all rows stay below the largest value that a row has, so an output that
// is finite comes out finite. What that costs are the last k bits of outputs near
// fp32's smallest. A value that is infinite stays so: the second term of a product of
// its own is never 0, and the merge adds none to an infinite first one.
//
// Splits leave (max, sum, accumulator) in the workspace and a second launch joins
// them by log-sum-exp; a single split without weights writes its output itself.
// With weights every score goes to the workspace (4 bytes a row and query head)
// and the second launch turns it into exp(s - lse) once the sums are known.
//
// 64 x 8 x 32768 x 128 e4m3 in 16-row pages: 638 us, 6.75 TB/s (a read-only stream
// exceeds the measured copy rate), up to 737 us (5.84 TB/s) where the power cap lowers
// the SM clock: it is bound by memory at full clock only (650 instructions a tile and
// warp, half of the issue slots). 32 x 8 x 4097 x 128 fp16: 82 us, with weights 97-101
// (scores 2, second launch 10). 131071 e4m3 keys of one sequence with weights: 58-61
// us for 277 MB, 50 of them a single wave of CTAs, then the second launch. Three CTAs
// an SM with two stages a warp against two with three: 661-750 and 722-810 us.
#include <math.h>

#include <cmath>
#include <type_traits>

#include "cache.cuh"
#include "mma_sync.cuh"

namespace pa {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxSplit = 512;

template <int KIND, int D, int HT>
struct DecCfg {
  static constexpr int kCtas = HT <= 8 ? 3 : 2;   // per SM
  static constexpr int kDepth = HT <= 8 ? 2 : 3;  // stages per warp
  static constexpr int kEsz = cache_esz(KIND);
  static constexpr int kRowBytes = D * kEsz;                           // 64, 128 or 256
  static constexpr int kBoxBytes = kRowBytes < 128 ? kRowBytes : 128;  // swizzled unit of a row
  static constexpr int kTK = 4096 / kRowBytes;                         // rows per tile
  static constexpr int kTileBytes = 4096;
  static constexpr int kScaleOff = 2 * kTileBytes;
  static constexpr int kStageBytes = kScaleOff + (cache_8bit(KIND) ? 512 : 0);
  static constexpr int kRingBytes = kWarps * kDepth * kStageBytes;
  // Merge area (aliases the ring): per warp m[16], l[16], acc[G][D] (or 8 rows of D + 4).
  static constexpr int kMergeFloats = kWarps * 32 + kWarps * 16 * D;
  static_assert(kMergeFloats * 4 <= kRingBytes, "merge area fits the ring");
  static constexpr int kSmemBytes = kRingBytes + 128;

  // Byte offset of byte `byte` of row `row` in a tile: 128-byte units one after
  // another, 16-byte pieces permuted so that the fragment loads meet no bank twice.
  static __device__ __forceinline__ int off(int row, int byte) {
    const int bx = byte / kBoxBytes, b = byte % kBoxBytes;
    const int sw = kBoxBytes == 128 ? (row & 7) : ((row >> 1) & 3);
    return bx * (kTK * kBoxBytes) + row * kBoxBytes + (((b >> 4) ^ sw) << 4) + (b & 15);
  }
};

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
  float* ws_ml;      // [B*Hq][nsplit][2]: max (log2 units), sum
  float* ws_scores;  // [B*Hq][score_stride] in log2 units, with weights only
  int* status;
  int64_t score_stride;
  int32_t G, nsplit, chunk;
  int32_t direct;    // one split, no weights: the first launch writes the output
  uint32_t unit;     // bytes; divides every stride of the cache
  uint32_t u_page, u_head, u_key;  // the strides in units
  uint32_t u_scale_page;
  float scale_log2;
  float acc_scale;   // 2^-k of the running O^T
};

__device__ __forceinline__ int seq_len(const DecodeArgs& a, int b, bool report) {
  if (!a.lens) return a.c.max_len;
  const int n = a.lens[b];
  if (n >= 0 && n <= a.c.max_len) return n;
  if (report) atomicExch(a.status, kStatusBadSeqLen);
  return n < 0 ? 0 : a.c.max_len;
}

// The cache streams through the L2 once: evict-first leaves room for the scores.
__device__ __forceinline__ uint64_t stream_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint.L2::128B [%0], [%1], 16, %2;" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two transposed 16 x 16 byte blocks: lane i gives the address of row i % 16 of
// block i / 16. Thread (g, c) gets bytes of columns g (r0) and g + 8 (r1) of the
// first block, rows 4c..4c+3 in a word, and of the second in r2, r3.
__device__ __forceinline__ void ldsm_b8_t(const void* p, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(smem_u32(p)));
}

// Four 8-bit codes a word, made ready for cvt2 (int8 becomes its value + 128).
template <int KIND>
__device__ __forceinline__ uint32_t prep8(uint32_t w) {
  return KIND == kCacheI8 ? w ^ 0x80808080u : w;
}
// The low (HI = 0) or high two codes of a prepared word as f16x2, exactly: int8
// through 1024 + u, whose last mantissa bit is worth 1.
template <int KIND, int HI>
__device__ __forceinline__ uint32_t cvt2(uint32_t w) {
  if (KIND == kCacheE4M3) {
    uint32_t h;
    if (HI)
      asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, u;\n\t}" : "=r"(h) : "r"(w));
    else
      asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(h) : "r"(w));
    return h;
  }
  const uint32_t u = byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(1152.f, 1152.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two floats as 16-bit values, cut off instead of rounded, the first in the low half.
template <bool BF16>
__device__ __forceinline__ uint32_t pack_cut(float lo, float hi) {
  if (BF16) return byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
  uint32_t d;
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

template <bool QBF16>
__device__ __forceinline__ void store_out(const DecodeArgs& a, int64_t i, float o) {
  if (QBF16)
    static_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(o);
  else
    static_cast<__half*>(a.out)[i] = __float2half_rn(o);
}

// log2 of a softmax denominator 2^M * L (L = 0: no keys; NaN stays NaN).
__device__ __forceinline__ float lse_of(float M, float L) {
  return L > 0.f ? M + log2f(L) : (L == 0.f ? -INFINITY : L);
}

template <int KIND, int D, bool QBF16, int HT>
__global__ void __launch_bounds__(kThreads, DecCfg<KIND, D, HT>::kCtas) cache_decode_kernel(const DecodeArgs a) {
  using C = DecCfg<KIND, D, HT>;
  constexpr int kDepth = C::kDepth;
  constexpr bool kF8 = cache_8bit(KIND);
  constexpr bool kMmaBf16 = KIND == kCacheBF16;
  constexpr bool kTwo = HT == 16;
  constexpr bool kSide = HT == 4;  // second terms in columns 4 to 7
  constexpr float kPScale = kMmaBf16 ? 0.03125f : 32768.f;
  constexpr uint32_t kCut = kMmaBf16 ? 0xffff0000u : 0xffffe000u;  // what 16 bits hold of an fp32
  constexpr int TK = C::kTK;
  constexpr int KS = D / 16;   // k-steps of Q K^T
  constexpr int MT = D / 16;   // m-tiles of V^T P^T
  constexpr int NT = TK / 8;   // n-tiles of Q K^T
  constexpr int PS = TK / 16;  // k-steps of V^T P^T
  extern __shared__ __align__(128) uint8_t smem[];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % a.nsplit;
  const int pair = blockIdx.x / a.nsplit;
  const int b = pair / a.c.Hkv, h = pair % a.c.Hkv;
  const int G = a.G;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // The length and the first pages are asked for together: table entries behind
  // the length are read but not used.
  const int k0 = split * a.chunk;  // below max_len
  const int k_most = a.chunk < a.c.max_len - k0 ? k0 + a.chunk : a.c.max_len;
  constexpr int RL = TK > 32 ? 2 : 1;  // rows of a tile per lane
  auto tile_row = [&](int j) { return k0 + (warp + kWarps * j) * TK; };
  // Pages of this lane's rows of own tile j (-1 where there can be none).
  auto load_pages = [&](int j, int32_t (&pg)[RL]) {
#pragma unroll
    for (int i = 0; i < RL; ++i) {
      const int r = tile_row(j) + lane + 32 * i;
      pg[i] = -1;
      if (lane + 32 * i < TK && r < k_most) {
        pg[i] = b;
        if (a.table) pg[i] = a.table[static_cast<int64_t>(b) * a.c.max_pages + fast_div(a.c.by_page, r)];
      }
    }
  };
  int32_t pg_next[RL];
  load_pages(0, pg_next);
  const int len = seq_len(a, b, threadIdx.x == 0 && split == 0 && h == 0);
  const int k1 = k_most < len ? k_most : (k0 < len ? len : k0);
  const int ntiles = (k1 - k0 + TK - 1) / TK;
  const int n_own = ntiles > warp ? (ntiles - warp + kWarps - 1) / kWarps : 0;
  const int64_t q0 = static_cast<int64_t>(b) * a.c.Hq + static_cast<int64_t>(h) * G;
  uint8_t* ring = smem + warp * (kDepth * C::kStageBytes);
  const uint32_t ring_u = smem_u32(ring);

  // ------------------------------------------------------------- loading
  // Row offsets travel between lanes as 32-bit counts of a.unit.
  constexpr int CPR = C::kRowBytes / 16;  // 16-byte pieces per row; a lane always takes the same one
  const uint8_t* const k_lane = a.k + (lane % CPR) * 16;
  const uint8_t* const v_lane = a.v + (lane % CPR) * 16;
  const float* const ks_head = kF8 ? a.ks + h * a.c.scale_head : nullptr;
  const float* const vs_head = kF8 ? a.vs + h * a.c.scale_head : nullptr;
  const uint64_t policy = stream_policy();
  auto issue = [&](int j, const int32_t (&pg)[RL]) {
    if (j < n_own) {
      const uint32_t st = ring_u + (j % kDepth) * C::kStageBytes;
      uint32_t off[RL];
      bool ok[RL], all = true;
#pragma unroll
      for (int i = 0; i < RL; ++i) {
        const int r = tile_row(j) + lane + 32 * i;
        const bool mine = lane + 32 * i < TK;
        ok[i] = mine && r < k1;
        if (ok[i] && a.table && (pg[i] < 0 || pg[i] >= a.c.num_pages)) {
          atomicExch(a.status, kStatusBadPage);
          ok[i] = false;
        }
        const int at = ok[i] ? cache_at(a.c, r) : 0;
        const int32_t page = ok[i] ? pg[i] : 0;
        off[i] = static_cast<uint32_t>(page) * a.u_page + h * a.u_head + at * a.u_key;
        if (kF8 && mine) {
          const uint64_t so = static_cast<uint64_t>(static_cast<uint32_t>(page)) * a.u_scale_page + fast_div(a.c.by_block, at);
          const uint32_t sdst = st + C::kScaleOff + (lane + 32 * i) * 4;
          cp_async4(sdst, ks_head + so, ok[i] ? 4u : 0u);
          cp_async4(sdst + TK * 4, vs_head + so, ok[i] ? 4u : 0u);
        }
        all = all && (ok[i] || !mine);
      }
      if (__all_sync(0xffffffffu, all)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = i * (32 / CPR) + lane / CPR;
          const uint64_t o = static_cast<uint64_t>(__shfl_sync(0xffffffffu, off[RL > 1 ? i / 4 : 0], row & 31)) * a.unit;
          const uint32_t dst = st + C::off(row, (lane % CPR) * 16);
          cp_async16(dst, k_lane + o, policy);
          cp_async16(dst + C::kTileBytes, v_lane + o, policy);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const int row = i * (32 / CPR) + lane / CPR;
          const int hi = RL > 1 ? i / 4 : 0;
          const uint64_t o = static_cast<uint64_t>(__shfl_sync(0xffffffffu, hi ? off[RL - 1] : off[0], row & 31)) * a.unit;
          const uint32_t n = __shfl_sync(0xffffffffu, (hi ? ok[RL - 1] : ok[0]) ? 16 : 0, row & 31);
          const uint32_t dst = st + C::off(row, (lane % CPR) * 16);
          cp_async16_or_zero(dst, k_lane + o, n);
          cp_async16_or_zero(dst + C::kTileBytes, v_lane + o, n);
        }
      }
    }
    cp_async_commit();
  };
  // ----------------------------------------------------------- Q fragments
  // Thread (g, c) = (lane / 4, lane % 4) holds head rows g and g + 8. For 8-bit
  // caches the head-dim order is permuted per thread (a dot product does not see
  // it), and a bf16 query becomes fp16 after a power of two of its own head that
  // puts the head's largest element into [2^14, 2^15): heads of one group may differ
  // in magnitude by any factor, and elements down to 2^-28 of their head's largest
  // keep all their bits.
  const int g = lane >> 2, c = lane & 3;
  float sl2 = a.scale_log2, sl2_hi = a.scale_log2;  // of heads g and g + 8
  uint32_t qa[KS][2], qh[KS][2];
  {
    const uint32_t* qw = static_cast<const uint32_t*>(a.q) + q0 * (D / 2);
    auto frag = [&](int head, int s, int w) -> uint32_t {
      const int d = kF8 ? (D / 4) * c + 4 * s + 2 * w : 16 * s + 2 * c + 8 * w;
      return head < G ? qw[head * (D / 2) + d / 2] : 0u;
    };
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        qa[s][w] = frag(kSide ? g & 3 : g, s, w);
        qh[s][w] = kTwo ? frag(g + 8, s, w) : 0u;
      }
    if (QBF16 && kF8) {
      // One head, held by the four lanes of equal g; returns scale_log2 over its factor.
      auto to_f16 = [&](uint32_t (&f)[KS][2]) -> float {
        float mx = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const float2 x = cache_unpack<true>(f[s][w]);
            mx = cache_amax(cache_amax(mx, x.x), x.y);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int e = static_cast<int>(__float_as_uint(mx) >> 23) - 127;  // floor(log2(mx)) for normal values
        e = e < -100 ? -100 : e;
        const float qs = __int_as_float((127 + 14 - e) << 23);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const float2 x = cache_unpack<true>(f[s][w]);
            f[s][w] = pack_pair<false>(x.x * qs, x.y * qs);
          }
        return a.scale_log2 * __int_as_float((127 - 14 + e) << 23);
      };
      sl2 = to_f16(qa);
      if (kTwo) sl2_hi = to_f16(qh);
    }
  }

  // --------------------------------------------------------------- compute
  float o[MT][4], o2[MT][4];  // O^T of heads 2c, 2c + 1 and (16-row tiles) 8 + those
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[mt][i] = o2[mt][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f, m_run2 = -INFINITY, l_run2 = 0.f;

  const uint32_t side_mask = g < 4 ? 0u : kCut;  // which term this lane gives
  // This thread's place in its head's scores, for own tile 0.
  float* const scores = a.ws_scores + (q0 + g) * a.score_stride + tile_row(0) + (kF8 ? 4 : 2) * c;
  // Rounds -kDepth..-1 only fill the stages: one copy of the code, which a short
  // call runs from a cold instruction cache.
#pragma unroll 1
  for (int j = -kDepth; j < n_own; ++j) {
    int32_t pg[RL];
#pragma unroll
    for (int i = 0; i < RL; ++i) pg[i] = pg_next[i];
    load_pages(j + kDepth + 1, pg_next);
    if (j < 0) {
      issue(j + kDepth, pg);
      continue;
    }
    cp_async_wait<kDepth - 1>();
    __syncwarp();
    const uint8_t* kt = ring + (j % kDepth) * C::kStageBytes;
    const uint8_t* vt = kt + C::kTileBytes;
    const int row0 = tile_row(j);
    const int rem = k1 - row0 < TK ? k1 - row0 : TK;

    // ---- S = Q K^T. Column n of n-tile nt is key 8 nt + n, or in 8 bits key
    // 16 (nt / 2) + 4 (n / 2) + 2 (nt % 2) + n % 2: a thread's columns of two
    // n-tiles are then the four keys 4c..4c+3 that it gets of V.
    float sacc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      sacc[nt][0] = sacc[nt][1] = sacc[nt][2] = sacc[nt][3] = 0.f;
      if (kF8) {
        const int row = 16 * (nt >> 1) + 4 * (g >> 1) + 2 * (nt & 1) + (g & 1);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint4 u = *reinterpret_cast<const uint4*>(kt + C::off(row, (D / 4) * c + 16 * i));
          const uint32_t w[4] = {prep8<KIND>(u.x), prep8<KIND>(u.y), prep8<KIND>(u.z), prep8<KIND>(u.w)};
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int s = 4 * i + t;
            mma16816<kMmaBf16>(sacc[nt], qa[s][0], qh[s][0], qa[s][1], qh[s][1], cvt2<KIND, 0>(w[t]),
                               cvt2<KIND, 1>(w[t]));
          }
        }
      } else {
        const int row = 8 * nt + (lane & 7);
#pragma unroll
        for (int s2 = 0; s2 < KS / 2; ++s2) {
          uint32_t b0, b1, b2, b3;
          ldsm_x4(kt + C::off(row, (4 * s2 + (lane >> 3)) * 16), b0, b1, b2, b3);
          mma16816<kMmaBf16>(sacc[nt], qa[2 * s2][0], qh[2 * s2][0], qa[2 * s2][1], qh[2 * s2][1], b0, b1);
          mma16816<kMmaBf16>(sacc[nt], qa[2 * s2 + 1][0], qh[2 * s2 + 1][0], qa[2 * s2 + 1][1], qh[2 * s2 + 1][1],
                             b2, b3);
        }
      }
    }

    // ---- softmax of the tile: keys key_of(nt, e) of heads g (columns 0-1), g + 8 (2-3)
    auto key_of = [&](int nt, int e) { return kF8 ? 16 * (nt >> 1) + 4 * c + 2 * (nt & 1) + e : 8 * nt + 2 * c + e; };
    float vw[NT][2];      // value scale over the power of two of the tile's largest, times 2^14
    float vtile = a.acc_scale / kPScale;
    if (kF8) {
      const float* sc = reinterpret_cast<const float*>(kt + C::kScaleOff);
      float vmax = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; nt += 2) {
        const float4 fk = *reinterpret_cast<const float4*>(sc + 8 * nt + 4 * c);
        const float4 fv = *reinterpret_cast<const float4*>(sc + TK + 8 * nt + 4 * c);
        const float k4[4] = {fk.x * sl2, fk.y * sl2, fk.z * sl2, fk.w * sl2};
        const float k4_hi[4] = {fk.x * sl2_hi, fk.y * sl2_hi, fk.z * sl2_hi, fk.w * sl2_hi};
        const float v4[4] = {fv.x, fv.y, fv.z, fv.w};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sacc[nt + u][e] *= k4[2 * u + e];
            if (kTwo) sacc[nt + u][2 + e] *= (QBF16 ? k4_hi : k4)[2 * u + e];
            vw[nt + u][e] = v4[2 * u + e];
            vmax = fmaxf(vmax, fabsf(v4[2 * u + e]));
          }
      }
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 1));
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));
      // Scales below 2^-112 stay as far below the factor as they are.
      const uint32_t e = max(__float_as_uint(vmax) >> 23, 15u);
      const float r = __uint_as_float((2u * 127u + 14u - e) << 23);
      vtile = __uint_as_float((e - 14u) << 23) * a.acc_scale;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        vw[nt][0] *= r;
        vw[nt][1] *= r;
      }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sacc[nt][e] *= sl2;
        vw[nt][0] = vw[nt][1] = kPScale;
      }
    }
    if (a.weights) {
      // Rows of a tile behind the length land in the padding of their head's scores.
      float* p0 = scores + static_cast<int64_t>(j) * (kWarps * TK);
#pragma unroll
      for (int u = 0; u < (kTwo ? 2 : 1); ++u) {
        if (g + 8 * u >= G) continue;
        float* p = p0 + u * 8 * a.score_stride;
#pragma unroll
        for (int nt = 0; nt < NT; nt += 2) {
          if (kF8) {
            __stcg(reinterpret_cast<float4*>(p + 8 * nt),
                   make_float4(sacc[nt][2 * u], sacc[nt][2 * u + 1], sacc[nt + 1][2 * u], sacc[nt + 1][2 * u + 1]));
          } else {
            __stcg(reinterpret_cast<float2*>(p + 8 * nt), make_float2(sacc[nt][2 * u], sacc[nt][2 * u + 1]));
            __stcg(reinterpret_cast<float2*>(p + 8 * nt + 8), make_float2(sacc[nt + 1][2 * u], sacc[nt + 1][2 * u + 1]));
          }
        }
      }
    }
    if (rem < TK) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key_of(nt, e & 1) >= rem) sacc[nt][e] = -INFINITY;
    }
    uint32_t pb[PS][2], pb2[PS][2];    // B fragments of P^T for the 16-key steps
    uint32_t pl[PS][2], pl2[PS][2];    // the second terms
    auto head_softmax = [&](int e0, float& m_h, float& l_h, uint32_t (&ph)[PS][2], uint32_t (&plo)[PS][2], float& alpha,
                            float& beta) {
      float mx = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mx = max3(mx, sacc[nt][e0], sacc[nt][e0 + 1]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float base = mx == -INFINITY ? 0.f : mx;
      float psum = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float p0 = ex2(sacc[nt][e0] - base), p1 = ex2(sacc[nt][e0 + 1] - base);
        psum += p0 + p1;
        float w0 = p0 * vw[nt][0], w1 = p1 * vw[nt][1];
        if (kSide) {  // this lane's term
          w0 -= __uint_as_float(__float_as_uint(w0) & side_mask);
          w1 -= __uint_as_float(__float_as_uint(w1) & side_mask);
        }
        ph[nt >> 1][nt & 1] = pack_cut<kMmaBf16>(w0, w1);
        if (!kSide) {
          const uint32_t u0 = __float_as_uint(w0), u1 = __float_as_uint(w1), more = kF8 ? 0u : 1u;  // never 0
          plo[nt >> 1][nt & 1] = pack_pair<kMmaBf16>(__uint_as_float(u0 | more) - __uint_as_float(u0 & kCut),
                                                     __uint_as_float(u1 | more) - __uint_as_float(u1 & kCut));
        }
      }
      const float m_new = fmaxf(m_h, mx);
      const float nb = m_new == -INFINITY ? 0.f : m_new;
      alpha = ex2(m_h - nb);
      beta = ex2(mx - nb);
      l_h = l_h * alpha + psum * beta;
      m_h = m_new;
      beta *= vtile;
    };
    float al, be, al2 = 1.f, be2 = 0.f;
    head_softmax(0, m_run, l_run, pb, pl, al, be);
    if (kTwo) head_softmax(2, m_run2, l_run2, pb2, pl2, al2, be2);
    const bool moved = __any_sync(0xffffffffu, al != 1.f || (kTwo && al2 != 1.f));

    // ---- O^T of the tile = V^T P^T
    float t[MT][4], t2[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) t[mt][i] = t2[mt][i] = 0.f;
#pragma unroll
    for (int sp = 0; sp < PS; ++sp) {
      const int kb = 16 * sp;
      if (kF8) {
#pragma unroll
        for (int mt = 0; mt < MT; mt += 2) {
          uint32_t r[4];
          ldsm_b8_t(vt + C::off(kb + (lane & 15), (mt + (lane >> 4)) * 16), r[0], r[1], r[2], r[3]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t x = prep8<KIND>(r[2 * u]), y = prep8<KIND>(r[2 * u + 1]);
            const uint32_t a0 = cvt2<KIND, 0>(x), a2 = cvt2<KIND, 1>(x), a1 = cvt2<KIND, 0>(y), a3 = cvt2<KIND, 1>(y);
            mma16816<kMmaBf16>(t[mt + u], a0, a1, a2, a3, pb[sp][0], pb[sp][1]);
            if (!kSide) mma16816<kMmaBf16>(t[mt + u], a0, a1, a2, a3, pl[sp][0], pl[sp][1]);
            if (kTwo) {
              mma16816<kMmaBf16>(t2[mt + u], a0, a1, a2, a3, pb2[sp][0], pb2[sp][1]);
              if (!kSide) mma16816<kMmaBf16>(t2[mt + u], a0, a1, a2, a3, pl2[sp][0], pl2[sp][1]);
            }
          }
        }
      } else {
        const int mm = lane >> 3;
        const int row = kb + 8 * (mm >> 1) + (lane & 7);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t a0, a1, a2, a3;
          ldsm_x4_t(vt + C::off(row, (2 * mt + (mm & 1)) * 16), a0, a1, a2, a3);
          mma16816<kMmaBf16>(t[mt], a0, a1, a2, a3, pb[sp][0], pb[sp][1]);
          if (!kSide) mma16816<kMmaBf16>(t[mt], a0, a1, a2, a3, pl[sp][0], pl[sp][1]);
          if (kTwo) {
            mma16816<kMmaBf16>(t2[mt], a0, a1, a2, a3, pb2[sp][0], pb2[sp][1]);
            if (!kSide) mma16816<kMmaBf16>(t2[mt], a0, a1, a2, a3, pl2[sp][0], pl2[sp][1]);
          }
        }
      }
    }
    __syncwarp();  // every lane has read this stage
    issue(j + kDepth, pg);

    // ---- join: heads 2c and 2c + 1 of the O^T columns this thread holds
    auto join = [&](float (&oo)[MT][4], const float (&tt)[MT][4], float alpha, float beta) {
      const float b0 = __shfl_sync(0xffffffffu, beta, 8 * c), b1 = __shfl_sync(0xffffffffu, beta, 8 * c + 4);
      if (moved) {
        const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * c), a1 = __shfl_sync(0xffffffffu, alpha, 8 * c + 4);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) oo[mt][i] *= (i & 1) ? a1 : a0;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) oo[mt][i] = fmaf(tt[mt][i], (i & 1) ? b1 : b0, oo[mt][i]);
    };
    join(o, t, al, be);
    if (kTwo) join(o2, t2, al2, be2);
  }
  cp_async_wait<0>();

  // ------------------------------------------------------- merge the warps
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
  l_run2 += __shfl_xor_sync(0xffffffffu, l_run2, 1);
  l_run2 += __shfl_xor_sync(0xffffffffu, l_run2, 2);
  __syncthreads();  // every stage has been used: the ring is free
  float* mw = reinterpret_cast<float*>(smem);  // [kWarps][16] max
  float* lw = mw + kWarps * 16;                // [kWarps][16] sum
  float* aw = lw + kWarps * 16;                // [kWarps][G][D], or [kWarps][8][kSideD]
  constexpr int kSideD = D + 4;                // four heads' stores meet no bank twice
  if (c == 0) {
    mw[warp * 16 + g] = m_run;
    lw[warp * 16 + g] = l_run;
    if (kTwo) {
      mw[warp * 16 + g + 8] = m_run2;
      lw[warp * 16 + g + 8] = l_run2;
    }
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int head = 2 * c + (i & 1), half = i >> 1;
      const int d = 16 * mt + 8 * half + g;
      if (kSide)
        aw[(warp * 8 + head) * kSideD + d] = o[mt][i];
      else if (head < G)
        aw[(warp * G + head) * D + d] = o[mt][i];
      if (kTwo && head + 8 < G) aw[(warp * G + head + 8) * D + d] = o2[mt][i];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += kThreads) {
    const int head = i / D, d = i % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, mw[w * 16 + head]);
    const float base = M == -INFINITY ? 0.f : M;
    float acc = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(mw[w * 16 + head] - base);
      float x;
      if (kSide) {  // an infinity has no second term
        x = aw[(w * 8 + head) * kSideD + d];
        const float rest = aw[(w * 8 + 4 + head) * kSideD + d];
        x += fabsf(x) < INFINITY ? rest : 0.f;
      } else {
        x = aw[(w * G + head) * D + d];
      }
      acc = fmaf(f, x, acc);
      L = fmaf(f, lw[w * 16 + head], L);
    }
    if (a.direct) {
      store_out<QBF16>(a, q0 * D + i, L == 0.f ? 0.f : acc / (L * a.acc_scale));
      if (a.lse && d == 0) a.lse[q0 + head] = lse_of(M, L) * kLn2;
      continue;
    }
    const int64_t slot = (q0 + head) * a.nsplit + split;
    a.ws_acc[slot * D + d] = acc;
    if (d == 0) {
      a.ws_ml[slot * 2] = M;
      a.ws_ml[slot * 2 + 1] = L;
    }
  }
}

// Second launch, started while the first one ends (it waits for its memory).
// grid.x = pairs (sequence, kv head). grid.y < out_ctas: joins the splits of E of
// the G x D outputs, thread (i, part) taking every kParts-th split (few splits:
// E = 256, one part; many: E = 32, eight parts). The other CTAs add the weights
// of kRowsPerCta rows, four a thread.
constexpr int kFinThreads = 256;
constexpr int kRowsPerCta = 4 * kFinThreads;
// E = 256 against E = 32: 8 splits with weights 10.6 and 12.7 us (5 x 8 x 1023 int8), 8
// to 16 without 8.4 and 8.4, 32 10.6 and 10.4, 55 14.5 and 12.6 (8 x 8192 e4m3).
constexpr int kFewSplits = 16;

template <int D, bool QBF16, int E>
__global__ void __launch_bounds__(kFinThreads) cache_finish_kernel(const DecodeArgs a) {
  constexpr int kParts = kFinThreads / E;
  constexpr int kHeads = E > D ? E / D : 1;  // heads of an output CTA
  constexpr int kMost = E == 32 ? kMaxSplit : kFewSplits;
  const int pair = blockIdx.x;
  const int b = pair / a.c.Hkv, h = pair % a.c.Hkv;
  const int64_t q0 = static_cast<int64_t>(b) * a.c.Hq + static_cast<int64_t>(h) * a.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ns = a.nsplit;
  const int out_ctas = (a.G * D + E - 1) / E;
  __shared__ float lse2[16];
  __shared__ float fac[kHeads * kMost];
  __shared__ float sums[kFinThreads];
  const int len = seq_len(a, b, false);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // log2 of head g's softmax denominator, by one warp.
  auto head_lse = [&](int g) -> float {
    const float2* ml = reinterpret_cast<const float2*>(a.ws_ml) + (q0 + g) * ns;
    float M = -INFINITY, L = 0.f;
    for (int s = lane; s < ns; s += 32) {
      const float2 x = ml[s];
      const float mn = fmaxf(M, x.x), base = mn == -INFINITY ? 0.f : mn;
      L = L * ex2(M - base) + x.y * ex2(x.x - base);
      M = mn;
    }
    const float top = warp_max(M), base = top == -INFINITY ? 0.f : top;
    L *= ex2(M - base);
#pragma unroll
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    return lse_of(top, L);
  };
  if (blockIdx.y < static_cast<unsigned>(out_ctas)) {
    const int i = blockIdx.y * E + threadIdx.x % E, part = threadIdx.x / E;
    const int g0 = blockIdx.y * E / D;
    const bool live = i < a.G * D;
    const int g = live ? i / D : a.G - 1, d = i % D;
    const float* acc = a.ws_acc + (q0 + g) * ns * D + d;
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = part + u * kParts < ns ? acc[(part + u * kParts) * D] : 0.f;
    if (warp < kHeads && g0 + warp < a.G) {
      const float z = head_lse(g0 + warp);
      const float* ml = a.ws_ml + (q0 + g0 + warp) * ns * 2;
      for (int s = lane; s < ns; s += 32) {
        const float ms = ml[2 * s];
        fac[warp * kMost + s] = ms == -INFINITY ? 0.f : ex2(ms - z) / a.acc_scale;
      }
      if (lane == 0 && a.lse && blockIdx.y * E % D == 0) a.lse[q0 + g0 + warp] = z * kLn2;
    }
    __syncthreads();
    const float* f = fac + (g - g0) * kMost;
    float o = 0.f;
    for (int s = part; s < ns; s += 8 * kParts) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s + u * kParts < ns) o = fmaf(f[s + u * kParts], x[u], o);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int n = s + (8 + u) * kParts;
        if (n < ns) x[u] = acc[static_cast<int64_t>(n) * D];
      }
    }
    if (kParts > 1) {
      sums[threadIdx.x] = o;
      __syncthreads();
#pragma unroll
      for (int p = 1; p < kParts; ++p) o += part == 0 ? sums[p * E + threadIdx.x % E] : 0.f;
    }
    if (part == 0 && live) store_out<QBF16>(a, q0 * D + i, o);
    return;
  }
  const int64_t r0 = static_cast<int64_t>(blockIdx.y - out_ctas) * kRowsPerCta;
  if (r0 >= len || (a.lens && a.lens[b] > a.c.max_len)) return;  // a wrong length: its weights stay
  const int64_t r = r0 + 4 * threadIdx.x;
  const float* sc = a.ws_scores + q0 * a.score_stride + r;
  float4 x[4];
#pragma unroll
  for (int g = 0; g < 4; ++g)
    x[g] = g < a.G && r < len ? *reinterpret_cast<const float4*>(sc + g * a.score_stride) : make_float4(0.f, 0.f, 0.f, 0.f);
  float* w = a.weights + b * a.c.row_seq + h * a.c.row_head + r;
  float old[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) old[e] = r + e < len ? w[e] : 0.f;
  for (int g = warp; g < a.G; g += kFinThreads / 32) {
    const float z = head_lse(g);
    if (lane == 0) lse2[g] = z;
  }
  __syncthreads();
  if (r >= len) return;
  for (int g0 = 0; g0 < a.G; g0 += 4) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (g0 + g >= a.G) break;
      const float z = lse2[g0 + g];
      if (z != -INFINITY) {
        old[0] += ex2(x[g].x - z);
        old[1] += ex2(x[g].y - z);
        old[2] += ex2(x[g].z - z);
        old[3] += ex2(x[g].w - z);
      }
      if (g0 + 4 + g < a.G) x[g] = *reinterpret_cast<const float4*>(sc + (g0 + 4 + g) * a.score_stride);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (r + e < len) w[e] = old[e];
}

struct DecodePlan {
  CacheView c;
  int G, nsplit, chunk;
  int64_t score_stride;
  bool weights, direct;
  uint32_t unit;
  size_t bytes;
};

// Splits of a (sequence, kv head). Where eight of each do not fill the resident
// CTAs, as many as do (one sequence of 131071 keys, 8 kv heads: 28 splits 78 us,
// 55 67, 74 78). Else up to eight, by a model of the launch in microseconds:
//   waves w = pairs * ns / resident CTAs; a last wave that fills a part f of the
//   slots still takes max(f, 0.75) of a full one (the reads saturate the memory
//   before all slots are taken), each wave costs its CTAs' start, merge and partial
//   results (6 us), the second launch 3 us, and a CTA reads 27 KB/us at most.
// Lengths are not known here; sequences shorter than max_len leave slots empty,
// which smaller chunks even out, so the largest count within 6 % is taken.
// Measured at 64 x 8 x 32768 x 128 e4m3: 1 split 838 us, 3 splits 679, 6 633; 16
// sequences: 2 splits 205, 3 176, 4 225; 64 ragged sequences of up to 8191 keys
// (int8, 2 kv heads of 64): 3 splits 37.3, 6 29.0.
int64_t choose_splits(int64_t pairs, int64_t tiles, int64_t wave, bool weights) {
  const int64_t most = tiles / kWarps < 1 ? 1 : tiles / kWarps;  // four tiles a CTA, one a warp
  if (pairs < 1) return 1;
  if (pairs * 8 < wave) {
    const int64_t ns = wave / pairs < most ? wave / pairs : most;
    return ns < kMaxSplit ? ns : kMaxSplit;
  }
  constexpr double kTileBytes = 8192, kBandwidth = 6.5e6, kCtaRate = 27e3;  // bytes, bytes/us
  const int64_t top = most < 8 ? most : 8;
  const double total = static_cast<double>(pairs) * tiles * kTileBytes / kBandwidth;
  double cost[9], least = 0;
  for (int64_t ns = 1; ns <= top; ++ns) {
    const double w = static_cast<double>(pairs * ns) / wave;
    const double full = std::floor(w), f = w - full;
    const double ineff = (full + (f > 1e-9 ? std::fmax(f, 0.75) : 0.0)) / w;
    const double chunk = static_cast<double>((tiles + ns - 1) / ns) * kTileBytes;
    cost[ns] = std::fmax(total * ineff, std::ceil(w) * chunk / kCtaRate) + 6.0 * std::ceil(w) + (ns > 1 || weights ? 3.0 : 0.0);
    least = ns == 1 ? cost[1] : std::fmin(least, cost[ns]);
  }
  int64_t ns = top;
  while (ns > 1 && cost[ns] > 1.06 * least) --ns;
  return ns;
}

pa_status plan_decode(const pa_block_cache_desc* d, bool paged, bool weights, DecodePlan* p) {
  *p = DecodePlan{};
  PA_TRY(check_cache(d, {paged, weights, true}, &p->c, "cache decode"));
  p->G = p->c.Hq / p->c.Hkv;
  p->weights = weights;
  // The largest power of two that divides every stride: row offsets are 32-bit
  // counts of it (at least 16 bytes, so 64 GiB per array at least).
  int64_t unit = 16;
  while (unit < (1 << 20) && (p->c.key_stride | p->c.head_stride | p->c.page_stride) % (2 * unit) == 0) unit *= 2;
  p->unit = static_cast<uint32_t>(unit);
  const double span = static_cast<double>(p->c.num_pages - 1) * static_cast<double>(p->c.page_stride / unit) +
                      static_cast<double>(p->c.Hkv - 1) * static_cast<double>(p->c.head_stride / unit) +
                      static_cast<double>(p->c.page_size - 1) * static_cast<double>(p->c.key_stride / unit);
  if (cache_8bit(p->c.kind) && p->c.scale_page > 0xffffffffLL) return fail(PA_ERR_UNSUPPORTED, "cache decode: scale_page_stride too large");
  if (span > 4294967295.0)
    return fail(PA_ERR_UNSUPPORTED, "cache decode: the cache spans more than 2^32 units of its strides' common power of two");
  const int tk = 4096 / (p->c.D * (cache_8bit(p->c.kind) ? 1 : 2));
  const int64_t pairs = static_cast<int64_t>(p->c.B) * p->c.Hkv;
  const int64_t tiles = (static_cast<int64_t>(p->c.max_len) + tk - 1) / tk;
  const int64_t wave = (p->G <= 8 ? 3 : 2) * static_cast<int64_t>(sm_count());
  int64_t ns = choose_splits(pairs, tiles, wave, weights);
  const int64_t per = (tiles + ns - 1) / ns;
  const int64_t chunk = per * tk;
  p->chunk = static_cast<int>(chunk < tk ? tk : chunk);
  ns = (static_cast<int64_t>(p->c.max_len) + p->chunk - 1) / p->chunk;
  p->nsplit = static_cast<int>(ns < 1 ? 1 : ns);
  p->direct = p->nsplit == 1 && !weights;
  p->score_stride = (static_cast<int64_t>(p->c.max_len) + 63) / 64 * 64;  // whole tiles
  const size_t heads = static_cast<size_t>(p->c.B) * p->c.Hq;
  p->bytes = 16;
  if (!p->direct) p->bytes += heads * p->nsplit * (p->c.D + 2) * sizeof(float);
  if (weights) p->bytes += heads * p->score_stride * sizeof(float);
  if (pairs * p->nsplit > 0x7fffffffLL) return fail(PA_ERR_UNSUPPORTED, "cache decode: grid too large");
  if (weights && p->c.max_len > 65000LL * kRowsPerCta) return fail(PA_ERR_UNSUPPORTED, "cache decode: too many keys for weights");
  return PA_OK;
}

template <int KIND, int D, bool QBF16, int HT>
pa_status launch_decode_ht(const DecodePlan& p, const DecodeArgs& a, cudaStream_t st) {
  auto kern = cache_decode_kernel<KIND, D, QBF16, HT>;
  constexpr int smem = DecCfg<KIND, D, HT>::kSmemBytes;
  static uint64_t attr_set = 0;
  PA_TRY(set_smem_attr_once(reinterpret_cast<const void*>(kern), smem, &attr_set));
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.c.B) * p.c.Hkv * p.nsplit);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  PA_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  if (p.direct) return PA_OK;
  // The second launch may start while the first ends; it waits for its memory.
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(kFinThreads);
  cfg.dynamicSmemBytes = 0;
  const bool few = p.nsplit <= kFewSplits;
  const int e = few ? 256 : 32;
  cfg.gridDim = dim3(static_cast<unsigned>(p.c.B) * p.c.Hkv,
                     (p.G * D + e - 1) / e + (p.weights ? (p.c.max_len + kRowsPerCta - 1) / kRowsPerCta : 0));
  PA_CUDA(few ? cudaLaunchKernelEx(&cfg, cache_finish_kernel<D, QBF16, 256>, a)
              : cudaLaunchKernelEx(&cfg, cache_finish_kernel<D, QBF16, 32>, a));
  return PA_OK;
}

template <int KIND, int D, bool QBF16>
pa_status launch_decode(const DecodePlan& p, const DecodeArgs& a, cudaStream_t st) {
  // Head tile of 4 rows and their second terms (groups 1-4), 8 rows (5-8) or 16 (9-16).
  return p.G <= 4   ? launch_decode_ht<KIND, D, QBF16, 4>(p, a, st)
         : p.G <= 8 ? launch_decode_ht<KIND, D, QBF16, 8>(p, a, st)
                    : launch_decode_ht<KIND, D, QBF16, 16>(p, a, st);
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
  a.direct = p.direct;
  a.unit = p.unit;
  a.u_scale_page = static_cast<uint32_t>(p.c.scale_page);
  a.u_page = static_cast<uint32_t>(p.c.page_stride / p.unit);
  a.u_head = static_cast<uint32_t>(p.c.head_stride / p.unit);
  a.u_key = static_cast<uint32_t>(p.c.key_stride / p.unit);
  a.scale_log2 = static_cast<float>(desc->cache.scale * 1.4426950408889634);
  a.acc_scale = 1.f;
  for (int64_t rows = 1; rows < p.c.max_len; rows *= 2) a.acc_scale *= 0.5f;
  void* own = nullptr;
  if (!workspace) PA_TRY(scratch_alloc(&own, p.bytes, st));
  const size_t slots = p.direct ? 0 : static_cast<size_t>(p.c.B) * p.c.Hq * p.nsplit;
  a.ws_scores = static_cast<float*>(workspace ? workspace : own);
  a.ws_acc = a.ws_scores + (p.weights ? static_cast<size_t>(p.c.B) * p.c.Hq * p.score_stride : 0);
  a.ws_ml = a.ws_acc + slots * p.c.D;
  pa_status rc = p.c.D == 128 ? launch_decode_kind<128>(p, a, st) : launch_decode_kind<64>(p, a, st);
  scratch_free(own, st);
  return rc;
}
