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
// Two launches, the second started while the first ends (one where few rows can
// go). `select`: a (sequence, kv head) is one CTA, or a cluster of up to eight where
// there are few of them. Each thread holds eight or sixteen rows' keys in registers,
// four neighbours at a time so that a warp's reads are whole lines (longer shares are
// read again in rounds: over 16384 rows a CTA for every digit and every rank, three
// to six times in all). The threshold key is found by radix selection, digits of 11,
// 11 and 10 bits counted in shared memory (a cluster's CTAs add their counts into
// each other's memory); it stops as soon as a digit's rows are all taken. Ranks of
// ties, holes and sources are prefix sums over the threads. Holes and sources go to
// two lists in the workspace, and the per-row arrays are written. `move` carries the
// rows over: in 16 bits a warp takes 32 list entries. The call reads 8 bytes a row,
// writes 12 bytes a kept row and moves what must move.
//
// In 8-bit caches a warp owns the keys or the values of a whole scale block, the
// one whose first hole is among the eight list entries it looks at; kept[] tells
// it what each place of the block gets, and it rescales the block by the rule of
// pa_cache_append. The block that `budget` cuts holds places below it and
// possibly sources at or above it: `select` puts its old scales aside, since
// `move` changes them while other warps read from it.
//
// One row over the budget of 2048 in 512 heads (e4m3): 14.7 us for 21.8 MB, nearly
// all latency (keys, the minimum, then the move's chain list -> block -> page and
// scale -> row), where no sequence can have more than eight rows to lose (max_seq_len
// <= budget + 8, and 2560 at most). Wider descriptors pay for their width: CTAs of
// max_seq_len rows, the keys of all of them read before the length is known, and a
// second launch with warps for as many moves as there could be: max_seq_len 4096
// 41.7 us, 8192 53.7, 32768 71.4 for the same row; 4097 rows to 4096 29.4. 128 heads
// of up to 8191 fp16 rows to 3001: 44 us for 137 MB (19 selection, 23 moves). 8 heads
// of 131071 int8 rows to 16384: 63 us for 71 MB (37 selection on the clusters' 64
// SMs, 26 moves, bound by look-ups and recoding).
#include <math.h>

#include "cache.cuh"

namespace pa {
namespace {

constexpr int kBins = 2048;     // digits of 11 bits (the last: 10)
constexpr int kScanThreads = 256;
constexpr int kMaxThreads = 1024;
constexpr int kMaxCluster = 8;  // portable cluster size
// Rows to evict that are picked one by one, about 2.7 us each for 512 heads of 2048
// rows, instead of by counting digits. One row: 14.7 us picked and moved by the same
// CTA, 22.9 by digits; eight 33.6 and 42.1. Where a second launch moves them (8192
// rows a head in the arrays): one row 53.7 and 70.2, eight 82.4 and 82.7, sixteen 113
// and 93.
constexpr int kFewRows = 8;

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
  int32_t* kept;     // [B][Hkv][budget]
  int32_t* holes;    // workspace [B][Hkv][list]
  int32_t* sources;  // workspace [B][Hkv][list]
  int32_t* counts;   // workspace [B][Hkv]: moves
  float* cut_scale;  // workspace [B][Hkv][2]: old scales of the cut block
  int* status;
  int32_t budget, recent, sinks, list;
  int32_t cluster;   // CTAs per (sequence, kv head)
  int32_t vec, vec_kept;  // the per-row arrays, kept[] can be used 16 bytes at a time
  int32_t by_block;  // 8 bits: `move` has a warp for every block below the budget
};

// Monotonic key of a weight; -0 counts as 0, NaN as the lowest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}
__device__ __forceinline__ int cluster_load(const int* p, uint32_t rank) {
  uint32_t at;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ void cluster_add(int* p, uint32_t rank, int v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("red.relaxed.cluster.shared::cluster.add.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

struct EvictShared {
  int hist[3][kBins];  // counts of the (sequence, kv head), one array a pass
  int own[kBins];      // clusters: this CTA's counts of the pass
  int warp_sum[2][32];
  int total[2];        // this CTA's ranks, read by its cluster
  int digit, left, all;
  int bad;             // clusters: warps that found a page out of range
  int found[32];       // this CTA's
};

// Ranks of the rows that a mask marks (bit i: row i of this thread, group i / 4
// being 128 rows of the warp, four a lane), in row order.
struct RowRank {
  uint32_t before, all;  // per group, a byte each: marks of the lanes before, of the warp
  int base;              // marks of the warps before
  template <int kGroups>
  __device__ __forceinline__ void count(uint32_t mask) {
    uint32_t p = 0;
#pragma unroll
    for (int q = 0; q < kGroups; ++q) p |= static_cast<uint32_t>(__popc(mask >> (4 * q) & 15u)) << (8 * q);
    uint32_t s = p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
      if (static_cast<int>(threadIdx.x & 31) >= o) s += y;
    }
    before = s - p;  // at most 128 in a byte: nothing carries over
    all = __shfl_sync(0xffffffffu, s, 31);
  }
  __device__ __forceinline__ int warp_total() const {
    return (all & 255u) + (all >> 8 & 255u) + (all >> 16 & 255u) + (all >> 24);
  }
  // Rank of the first row of group q.
  __device__ __forceinline__ int group(int q) const {
    int r = base + (before >> (8 * q) & 255u);
    for (int i = 0; i < q; ++i) r += all >> (8 * i) & 255u;
    return r;
  }
};

// Exclusive prefix sum over the CTA's threads; `total` receives the sum.
__device__ __forceinline__ int cta_scan(int x, int* warp_sum, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();  // earlier readers of warp_sum are done
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  int w = lane < warps ? warp_sum[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return (warp > 0 ? before : 0) + s - x;
}

// Sums of x and y over the warps before this one, and over all of them.
__device__ __forceinline__ int4 warps_before(int x, int y, int (*warp_sum)[32]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  __syncthreads();  // earlier readers of warp_sum are done
  if (lane == 0) {
    warp_sum[0][warp] = x;
    warp_sum[1][warp] = y;
  }
  __syncthreads();
  const int u = lane < warps ? warp_sum[0][lane] : 0, v = lane < warps ? warp_sum[1][lane] : 0;
  return make_int4(__reduce_add_sync(0xffffffffu, lane < warp ? u : 0), __reduce_add_sync(0xffffffffu, lane < warp ? v : 0),
                   __reduce_add_sync(0xffffffffu, u), __reduce_add_sync(0xffffffffu, v));
}

// 16 codes of scale s as codes of scale `to`: code * s / to, rounded once more.
template <int KIND>
__device__ __forceinline__ uint4 recode_easy(const uint4& q, float s, float to) {
  const __half2 r = cache_ratio(s, to);
  return make_uint4(cache_rescale4<KIND>(q.x, r), cache_rescale4<KIND>(q.y, r), cache_rescale4<KIND>(q.z, r),
                    cache_rescale4<KIND>(q.w, r));
}
template <int KIND>
__device__ __noinline__ uint4 recode(uint4 q, float s, float to) {
  if (s == to) return q;
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t o[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 f = cache_dec2<KIND>(w[e >> 1] >> (16 * (e & 1)));
    o[e >> 1] |= cache_enc2<KIND>(__fdiv_rn(f.x * s, to), __fdiv_rn(f.y * s, to)) << (16 * (e & 1));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// What a warp needs of up to 32 moves into a block.
struct MoveSlot {
  int64_t from;  // source row, bytes from the cache's base
  float scale;   // the source's scale
  int place;     // row in the block
};
constexpr int kMoveWarps = 8;

// Moves into the scale block of rows lo.. of a cache's keys or values, by one
// warp; src0 is kept[lo + lane] (or lo + lane behind the block). Places are taken
// 32 at a time: lane i looks up place i's source, and the
// moves among them are packed into `slots` (the warp's own shared memory), so that
// rows that stay cost no lanes. Rows are then read in steps of four rounds; a
// block of one step stays in registers between the maximum and the coding, larger
// ones are read again.
template <int KIND, int D>
__device__ __forceinline__ void move_block(const EvictArgs& a, int kv, int b, int h, int64_t pair, int lo, int src0,
                                           MoveSlot* slots) {
  constexpr int kPieces = D / 16;      // lanes per row
  constexpr int kRows = 32 / kPieces;  // rows per round of a warp
  constexpr int kStep = 4 * kRows;     // rows per step: 16 or 32
  const int lane = threadIdx.x & 31;
  const int bs = a.c.scale_block, n = a.budget;
  const int hi = n - lo > bs ? lo + bs : n;
  const int cut = n % bs ? n / bs : -1;  // the block whose old scales were put aside
  const int ch = (lane % kPieces) * 16;
  const int32_t* kept = a.kept + pair * n;
  uint8_t* cache = kv ? a.cache[1] : a.cache[0];
  float* scales = kv ? a.scales[1] : a.scales[0];
  const int32_t page = cache_page(a.c, a.table, b, lo, a.status);
  if (page < 0) return;
  const int at_lo = cache_at(a.c, lo);
  float* const sp = scales + cache_scale(a.c, page, h, at_lo);
  uint8_t* const dst0 = cache + cache_row(a.c, page, h, at_lo) + ch;
  const float was = *sp;
  bool stays = false;  // some place keeps its row
  // Packs the moves of the 32 places from `first` on; returns their number.
  auto look_up = [&](int first) -> int {
    const int r = first + lane;
    const int src = first == lo ? src0 : r < hi ? kept[r] : r;
    MoveSlot m{-1, 0.f, r - lo};
    if (src != r) {
      const int32_t ps = cache_page(a.c, a.table, b, src, a.status);
      if (ps >= 0) {
        const int at = cache_at(a.c, src);
        m.from = cache_row(a.c, ps, h, at);
        m.scale = src / bs == cut ? a.cut_scale[pair * 2 + kv] : scales[cache_scale(a.c, ps, h, at)];
      }
    }
    const uint32_t moves = __ballot_sync(0xffffffffu, m.from >= 0);
    stays = stays || __any_sync(0xffffffffu, r < hi && src == r);
    __syncwarp();  // the slots' last readers are done
    if (m.from >= 0) slots[__popc(moves & ((1u << lane) - 1u))] = m;
    __syncwarp();
    return __popc(moves);
  };
  uint4 x[4];
  float s[4];
  int place[4];  // -1: nothing
  auto read = [&](int first, int count) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = first + u * kRows + lane / kPieces;
      x[u] = make_uint4(0u, 0u, 0u, 0u);
      s[u] = 0.f;
      place[u] = -1;
      if (j < count) {
        const MoveSlot m = slots[j];
        x[u] = *reinterpret_cast<const uint4*>(cache + m.from + ch);
        s[u] = m.scale;
        place[u] = m.place;
      }
    }
  };
  float amax = 0.f;
  int count = 0;
  for (int first = lo; first < hi; first += 32) {
    count = look_up(first);
    for (int i = 0; i < count; i += kStep) {
      read(i, count);
#pragma unroll
      for (int u = 0; u < 4; ++u) amax = cache_amax(amax, cache_absmax<KIND>(x[u]) * s[u]);
    }
  }
  const float need = cache_need_scale<KIND>(warp_max(amax));
  const float old = stays ? was : 0.f;
  const float to = old > need ? old : need;
  const bool again = hi - lo > 32 || count > kStep;
  for (int first = lo; first < hi; first += 32) {
    if (hi - lo > 32) count = look_up(first);
    for (int i = 0; i < count; i += kStep) {
      if (again) read(i, count);
      bool easy = true;
#pragma unroll
      for (int u = 0; u < 4; ++u) easy = easy && (place[u] < 0 || cache_easy_ratio(s[u], to));
      if (__all_sync(0xffffffffu, easy)) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (place[u] >= 0)
            *reinterpret_cast<uint4*>(dst0 + place[u] * a.c.key_stride) = recode_easy<KIND>(x[u], s[u], to);
      } else {
#pragma unroll 1
        for (int u = 0; u < 4; ++u) {
          const int p = u == 0 ? place[0] : u == 1 ? place[1] : u == 2 ? place[2] : place[3];
          const float f = u == 0 ? s[0] : u == 1 ? s[1] : u == 2 ? s[2] : s[3];
          const uint4 q = u == 0 ? x[0] : u == 1 ? x[1] : u == 2 ? x[2] : x[3];
          if (p >= 0) *reinterpret_cast<uint4*>(dst0 + p * a.c.key_stride) = recode<KIND>(q, f, to);
        }
      }
    }
  }
  if (stays && to != old)
    for (int r = lo + lane / kPieces; r < hi; r += kRows) {
      if (kept[r] != r) continue;
      uint4* p = reinterpret_cast<uint4*>(dst0 + (r - lo) * a.c.key_stride);
      *p = cache_easy_ratio(old, to) ? recode_easy<KIND>(*p, old, to) : recode<KIND>(*p, old, to);
    }
  __syncwarp();
  if (lane == 0) *sp = to;
}

// List entries a warp takes at a time.
constexpr int move_entries(int kind) { return cache_8bit(kind) ? 8 : 32; }

// Moves by list entries, by one warp: in 16 bits the rows of 32 entries; in 8 bits
// the scale blocks, of the keys or the values, whose first hole is among eight
// entries (more warps than blocks: the chain of look-ups is what takes the time).
template <int KIND, int D>
__device__ __forceinline__ void move_entries_of(const EvictArgs& a, int64_t pair, int b, int h, int chunk, int kv,
                                                int m, MoveSlot* slots) {
  const int lane = threadIdx.x & 31;
  const int32_t* holes = a.holes + pair * a.list;
  const int k0 = chunk * move_entries(KIND), k = k0 + lane;
  const int cnt = m - k0 < move_entries(KIND) ? m - k0 : move_entries(KIND);
  if (cache_8bit(KIND)) {
    const int bs = a.c.scale_block;
    const int block = lane < cnt ? holes[k] / bs : -1;
    const int prev = lane < cnt && k > 0 ? holes[k - 1] / bs : -1;
    uint32_t leads = __ballot_sync(0xffffffffu, lane < cnt && block != prev);
    while (leads) {
      const int l = __ffs(leads) - 1;
      leads &= leads - 1;
      const int lo = __shfl_sync(0xffffffffu, block, l) * bs;
      const int r = lo + lane;
      const int src0 = lane < bs && r < a.budget ? a.kept[pair * a.budget + r] : r;
      move_block<KIND, D>(a, kv, b, h, pair, lo, src0, slots);
    }
    return;
  }
  constexpr int kPieces = D / 8;       // lanes per row
  constexpr int kRows = 32 / kPieces;  // rows per step of a warp
  int64_t from = -1, to = -1;
  if (lane < cnt) {
    const int dst = holes[k], src = a.sources[pair * a.list + k];
    const int32_t pd = cache_page(a.c, a.table, b, dst, a.status), ps = cache_page(a.c, a.table, b, src, a.status);
    if (pd >= 0 && ps >= 0) {
      to = cache_row(a.c, pd, h, cache_at(a.c, dst));
      from = cache_row(a.c, ps, h, cache_at(a.c, src));
    }
  }
  const int ch = (lane % kPieces) * 16;
  for (int i = 0; i < cnt; i += 4 * kRows) {
    uint4 x[4][2];
    int64_t d[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = i + u * kRows + lane / kPieces;
      const int64_t s = __shfl_sync(0xffffffffu, from, j & 31);
      d[u] = __shfl_sync(0xffffffffu, to, j & 31);
      if (j >= cnt) d[u] = -1;
      if (d[u] >= 0) {
        x[u][0] = *reinterpret_cast<const uint4*>(a.cache[0] + s + ch);
        x[u][1] = *reinterpret_cast<const uint4*>(a.cache[1] + s + ch);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (d[u] >= 0) {
        *reinterpret_cast<uint4*>(a.cache[0] + d[u] + ch) = x[u][0];
        *reinterpret_cast<uint4*>(a.cache[1] + d[u] + ch) = x[u][1];
      }
  }
}

// kThreads and kCtas bound the registers: 1024 threads, or four CTAs of 256 to 320
// for many short sequences, so that 512 of them run at once.
// kMoveKind >= 0: at most kFewRows rows go, and the CTA carries the rows over too
// (the rest of the kernel is then not reached, which the compiler would report).
#pragma nv_diagnostic push
#pragma nv_diag_suppress 128
template <int kKeys, int kThreads, int kCtas, int kMoveKind, int kMoveD>
__global__ void __launch_bounds__(kThreads, kCtas) cache_select_kernel(const EvictArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  EvictShared& sh = *reinterpret_cast<EvictShared*>(smem_raw);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int C = a.cluster;
  const int rank = blockIdx.x % C;
  const int64_t pair = blockIdx.x / C;
  const int h = static_cast<int>(pair % a.c.Hkv), b = static_cast<int>(pair / a.c.Hkv);
  const int tid = threadIdx.x, T = blockDim.x;
  const int n = a.budget;
  int len = a.lens[b];
  const int32_t* pos = a.positions ? a.positions + b * a.c.row_seq + h * a.c.row_head : nullptr;
  const float* w = a.weights + b * a.c.row_seq + h * a.c.row_head;
  float* w_out = a.weights_out ? a.weights_out + b * a.c.row_seq + h * a.c.row_head : nullptr;
  int32_t* p_out = a.positions_out ? a.positions_out + b * a.c.row_seq + h * a.c.row_head : nullptr;
  int32_t* kept = a.kept + pair * n;
  int32_t* holes = a.holes + pair * a.list;
  int32_t* sources = a.sources + pair * a.list;
  constexpr int kGroups = kKeys / 4;
  const int lane = tid & 31;
  const int per_round = T * kKeys;
  // A thread's rows of a round: group q is four rows from my_row + 128 q on.
  int64_t my_row = 0;
  float4 wv[kGroups];
  int4 pv[kGroups];
  auto fetch = [&](int64_t first, int64_t end) {
    my_row = first + (tid >> 5) * (32 * kKeys) + lane * 4;
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      const int64_t r = my_row + q * 128;
      const int r32 = static_cast<int>(r);
      wv[q] = make_float4(0.f, 0.f, 0.f, 0.f);
      pv[q] = make_int4(r32, r32 + 1, r32 + 2, r32 + 3);
      if (r + 4 <= end && a.vec) {
        wv[q] = *reinterpret_cast<const float4*>(w + r);
        if (pos) pv[q] = *reinterpret_cast<const int4*>(pos + r);
      } else if (r < end) {
        wv[q].x = w[r];
        if (r + 1 < end) wv[q].y = w[r + 1];
        if (r + 2 < end) wv[q].z = w[r + 2];
        if (r + 3 < end) wv[q].w = w[r + 3];
        if (pos) {
          pv[q].x = pos[r];
          if (r + 1 < end) pv[q].y = pos[r + 1];
          if (r + 2 < end) pv[q].z = pos[r + 2];
          if (r + 3 < end) pv[q].w = pos[r + 3];
        }
      }
    }
  };
  // One CTA's first rows, and a page to look at for each thread, do not depend on the
  // length: asked for together with it.
  const int32_t my_page = C == 1 && a.table && tid < a.c.max_pages ? a.table[static_cast<int64_t>(b) * a.c.max_pages + tid] : 0;
  if (C == 1) fetch(0, a.c.max_len);
  const bool bad = len < 0 || len > a.c.max_len;
  if (h == 0 && rank == 0 && tid == 0) {
    if (bad) atomicExch(a.status, kStatusBadSeqLen);
    a.lens_out[b] = bad ? len : (len < n ? len : n);
  }
  if (bad) len = 0;
  if (len <= n) {  // nothing to evict (the whole cluster leaves here)
    if (rank == 0 && tid == 0) a.counts[pair] = 0;
    for (int64_t r = rank * T + tid; r < n; r += C * T) {
      kept[r] = r < len ? static_cast<int32_t>(r) : -1;
      if (r < len && w_out) w_out[r] = w[r];
      if (r < len && p_out) p_out[r] = pos ? pos[r] : static_cast<int32_t>(r);
    }
    return;
  }
  auto sync_all = [&]() {
    if (C > 1)
      cluster_sync();
    else
      __syncthreads();
  };
  // This CTA's rows: [row0, row_end), in rounds of T * kKeys.
  const int share = ((len + C - 1) / C + 3) / 4 * 4;
  const int64_t row0 = static_cast<int64_t>(rank) * share;
  const int64_t row_end = row0 + share < len ? row0 + share : len;
  const int rounds = (share + per_round - 1) / per_round;
  const int64_t next = a.next ? a.next[b] : len;
  const int64_t newest = next - a.recent;
  uint32_t keys[kKeys];
  uint32_t live = 0;  // rows this thread holds in the current round
  auto row_of = [&](int i) { return my_row + (i / 4) * 128 + (i & 3); };
  auto rank_keys = [&]() {
    live = 0;
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      const float wf[4] = {wv[q].x, wv[q].y, wv[q].z, wv[q].w};
      const int pf[4] = {pv[q].x, pv[q].y, pv[q].z, pv[q].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        live |= row_of(4 * q + e) < row_end ? 1u << (4 * q + e) : 0u;
        keys[4 * q + e] = pf[e] >= newest || pf[e] < a.sinks ? 0xffffffffu : weight_key(wf[e]);
      }
    }
  };
  auto load_keys = [&](int round) {
    fetch(row0 + static_cast<int64_t>(round) * per_round, row_end);
    rank_keys();
  };
  // kept[] below the budget as if every row stayed, and weights and positions too
  // (a cluster's few CTAs with such rows leave that to the end); places that
  // receive rows are written again.
  auto copy_rows = [&]() {
    const bool copy_w = C == 1 && w_out && w_out != w, copy_p = C == 1 && p_out && p_out != pos;
    const int64_t end = row_end < n ? row_end : n;
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      const int64_t r = my_row + q * 128;
      const int r32 = static_cast<int>(r);
      if (r + 4 <= end && a.vec) {
        if (copy_w) *reinterpret_cast<float4*>(w_out + r) = wv[q];
        if (copy_p) *reinterpret_cast<int4*>(p_out + r) = pv[q];
      } else {
        const float wf[4] = {wv[q].x, wv[q].y, wv[q].z, wv[q].w};
        const int pf[4] = {pv[q].x, pv[q].y, pv[q].z, pv[q].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (r + e < end && copy_w) w_out[r + e] = wf[e];
          if (r + e < end && copy_p) p_out[r + e] = pf[e];
        }
      }
      if (r + 4 <= end && a.vec_kept) {
        *reinterpret_cast<int4*>(kept + r) = make_int4(r32, r32 + 1, r32 + 2, r32 + 3);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r + e < end) kept[r + e] = r32 + e;
      }
    }
  };

  // Whether the warp found a page of the sequence out of range (a cluster's CTAs share
  // them out). The sequence is then left as it was; that is looked at when the lists
  // are complete, until when only copies of what it holds have been written.
  auto look_at_pages = [&]() {
    int wrong = 0;
    if (a.table) {
      const int used = fast_div(a.c.by_page, len - 1) + 1;
      if (C == 1) wrong = tid < used && (my_page < 0 || my_page >= a.c.num_pages);
#pragma unroll 1
      for (int i = rank * T + tid + (C == 1 ? T : 0); i < used; i += C * T) {
        const int32_t page = a.table[static_cast<int64_t>(b) * a.c.max_pages + i];
        wrong |= page < 0 || page >= a.c.num_pages;
      }
      if (wrong) atomicExch(a.status, kStatusBadPage);
      wrong = __any_sync(0xffffffffu, wrong);
    }
    if (lane == 0) sh.found[tid >> 5] = wrong;
  };
  auto leave = [&]() {
    if (h == 0 && rank == 0 && tid == 0) a.lens_out[b] = len;
    if (rank == 0 && tid == 0) a.counts[pair] = 0;
    for (int r = rank * T + tid; r < n; r += C * T) kept[r] = -1;
  };

  // ------------------------------------------------ threshold: radix selection
  // What `move` needs apart from the lists, by one thread or two.
  auto put_aside = [&](int moves) {
    if (rank == 0 && tid == 0) a.counts[pair] = moves;
    if (cache_8bit(a.c.kind) && rank == 0 && tid < 2 && n % a.c.scale_block) {
      const int32_t page = cache_page(a.c, a.table, b, n, a.status);
      a.cut_scale[pair * 2 + tid] = page < 0 ? 0.f : a.scales[tid][cache_scale(a.c, page, h, cache_at(a.c, n))];
    }
  };

  // ------------------------------------------- a few rows: one minimum at a time
  // The rows that go are the smallest keys, the highest row among equals; a budget
  // that is kept up every step evicts one. No digits are counted and no ranks
  // summed: the holes are the evicted rows below the budget, the sources the rows
  // behind it that were not evicted.
  if (C == 1 && rounds == 1 && len - n <= kFewRows) {
    rank_keys();
    copy_rows();
    look_at_pages();
    const int warp = tid >> 5, warps = T >> 5, out = len - n;
    for (int i = 0; i < out; ++i) {
      uint32_t key = 0xffffffffu;
      int row = -1;
#pragma unroll
      for (int k = 0; k < kKeys; ++k)
        if ((live >> k & 1u) && keys[k] <= key) {  // a thread's rows ascend
          key = keys[k];
          row = static_cast<int>(row_of(k));
        }
      const uint32_t wk = __reduce_min_sync(0xffffffffu, key);
      const int wr = __reduce_max_sync(0xffffffffu, key == wk ? row : -1);
      if (lane == 0) {
        sh.warp_sum[0][warp] = static_cast<int>(wk);
        sh.warp_sum[1][warp] = wr;
      }
      __syncthreads();
      const int r = lane < warps ? sh.warp_sum[1][lane] : -1;
      const uint32_t v = r >= 0 ? static_cast<uint32_t>(sh.warp_sum[0][lane]) : 0xffffffffu;
      const uint32_t least = __reduce_min_sync(0xffffffffu, v);
      const int gone = __reduce_max_sync(0xffffffffu, v == least ? r : -1);
#pragma unroll
      for (int k = 0; k < kKeys; ++k)
        if (row_of(k) == gone) live &= ~(1u << k);
      if (tid == 0) sh.own[i] = gone;
      __syncthreads();
    }
    if (__any_sync(0xffffffffu, lane < warps && sh.found[lane])) {
      leave();
      return;
    }
    if (tid < 32) {
      const int e = lane < out ? sh.own[lane] : 0x7fffffff;
      int before = 0, kept_before = 0;
      bool evicted = false;
      for (int i = 0; i < out; ++i) {
        const int x = sh.own[i];
        before += x < e;
        kept_before += x >= n && x < n + lane;
        evicted = evicted || x == n + lane;
      }
      if (e < n) sh.hist[0][before] = e;
      if (lane < out && !evicted) sh.hist[1][lane - kept_before] = n + lane;
      const int moves = __popc(__ballot_sync(0xffffffffu, e < n));
      __syncwarp();
      if (lane < moves) {
        const int d = sh.hist[0][lane], q = sh.hist[1][lane];
        holes[lane] = d;
        sources[lane] = q;
        kept[d] = q;
        if (w_out) w_out[d] = w[q];
        if (p_out) p_out[d] = pos ? pos[q] : q;
      }
      put_aside(moves);
      if (lane == 0) sh.left = moves;
    }
    if constexpr (kMoveKind >= 0) {
      __syncthreads();
      MoveSlot* const slots = reinterpret_cast<MoveSlot*>(&sh.hist[2][0]) + warp * 32;
      constexpr int kSides = cache_8bit(kMoveKind) ? 2 : 1;
      if (warp < kSides && sh.left > 0)
        move_entries_of<kMoveKind, kMoveD>(a, pair, b, h, 0, warp, sh.left, slots);
    }
    return;
  }
  if (kMoveKind >= 0) return;

  // A cluster's CTAs add into each other's arrays, so all are cleared up front.
  for (int i = tid; i < (C > 1 ? 4 : 1) * kBins; i += T) (&sh.hist[0][0])[i] = 0;  // own follows hist
  if (C > 1) fetch(row0, row_end);
  if (tid == 0) sh.bad = 0;
  rank_keys();
  copy_rows();
  look_at_pages();
  sync_all();
  uint32_t prefix = 0;
  int left = n;  // rows to take among those that match the prefix
  bool all = false;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const int width = pass == 2 ? 10 : 11;
#pragma unroll 1
    for (int round = 0; round < rounds; ++round) {
      if (pass > 0 ? rounds > 1 : round > 0) load_keys(round);
      if (pass == 0 && round > 0) copy_rows();
#pragma unroll
      for (int i = 0; i < kKeys; ++i)
        if ((live >> i & 1u) && (pass == 0 || (keys[i] >> (shift + width)) == (prefix >> (shift + width))))
          atomicAdd((C > 1 ? sh.own : sh.hist[pass]) + ((keys[i] >> shift) & ((1u << width) - 1u)), 1);
    }
    if (C > 1) {
      __syncthreads();
      for (int i = tid; i < kBins; i += T) {
        const int x = sh.own[i];
        if (x == 0) continue;
        sh.own[i] = 0;
        for (int q = 0; q < C; ++q) cluster_add(&sh.hist[pass][i], q, x);
      }
      if (pass == 0 && tid < T >> 5 && sh.found[tid])
        for (int q = 0; q < C; ++q) cluster_add(&sh.bad, q, 1);
    }
    sync_all();
    // Thread t < 256 takes bins 8 t' .. 8 t' + 7 from the top, t' = 255 - t.
    int bins[kBins / kScanThreads], sum = 0;
    if (C == 1 && pass < 2)
      for (int i = tid; i < kBins; i += T) sh.hist[pass + 1][i] = 0;
    if (tid < kScanThreads) {
      const int first = (kScanThreads - 1 - tid) * (kBins / kScanThreads);
#pragma unroll
      for (int i = 0; i < kBins / kScanThreads; ++i) {
        bins[i] = sh.hist[pass][first + i];
        sum += bins[i];
      }
    }
    int total;
    int above = cta_scan(sum, sh.warp_sum[0], &total);
    if (tid < kScanThreads && above < left && above + sum >= left) {
      const int first = (kScanThreads - 1 - tid) * (kBins / kScanThreads);
#pragma unroll
      for (int i = kBins / kScanThreads - 1; i >= 0; --i) {
        if (above < left && above + bins[i] >= left) {
          sh.digit = first + i;
          sh.left = left - above;
          sh.all = bins[i] == left - above;
        }
        above += bins[i];
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(sh.digit) << shift;
    left = sh.left;
    all = sh.all != 0;
    if (all) break;  // every row with this prefix is taken: no need to look further
  }

  // --------------------------------------------- ranks of ties, holes, sources
  // Kept: keys above the prefix, and of the keys that equal it the first `left`
  // (all keys from the prefix up, where `all`). Two sweeps: the counts of each
  // CTA, then, with the counts of the CTAs before it, the lists.
  // Sums of total[0] and total[1] over the CTAs before this one, and of total[0] over all.
  auto before = [&](const int* total) -> int4 {
    const int x = lane < C ? cluster_load(total, lane) : 0, y = lane < C ? cluster_load(total + 1, lane) : 0;
    return make_int4(__reduce_add_sync(0xffffffffu, lane < rank ? x : 0),
                     __reduce_add_sync(0xffffffffu, lane < rank ? y : 0), __reduce_add_sync(0xffffffffu, x), 0);
  };
  int tie_base = 0;
  if (!all) {
    int own = 0;
#pragma unroll 1
    for (int round = 0; round < rounds; ++round) {
      if (rounds > 1) load_keys(round);
#pragma unroll
      for (int i = 0; i < kKeys; ++i) own += (live >> i & 1u) && keys[i] == prefix;
    }
    if (C > 1) {
      int total;
      cta_scan(own, sh.warp_sum[0], &total);
      if (tid == 0) sh.total[0] = total;
      cluster_sync();
      tie_base = before(sh.total).x;
      cluster_sync();  // total is used again
    }
  }
  int hole_base = 0, src_base = 0, hole_all = 0;
  uint32_t keep = 0, hole = 0, src = 0;
  RowRank holes_at, src_at;
  int round_holes = 0, round_src = 0;
  // The current round's masks, and ranks inside it.
  auto rank_round = [&](int& ties) {
    keep = 0;
    uint32_t tie = 0;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      if (all ? keys[i] >= prefix : keys[i] > prefix) keep |= 1u << i;
      if (!all && keys[i] == prefix) tie |= 1u << i;
    }
    keep &= live;
    tie &= live;
    if (!all) {
      RowRank at;
      at.count<kGroups>(tie);
      const int4 sum = warps_before(at.warp_total(), 0, sh.warp_sum);
      at.base = ties + sum.x;
      ties += sum.z;
#pragma unroll
      for (int q = 0; q < kGroups; ++q) {
        int r = at.group(q);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (tie >> (4 * q + e) & 1u) {
            if (r < left) keep |= 1u << (4 * q + e);
            ++r;
          }
      }
    }
    uint32_t low = 0;  // rows below the budget
#pragma unroll
    for (int i = 0; i < kKeys; ++i) low |= row_of(i) < n ? 1u << i : 0u;
    hole = ~keep & live & low;
    src = keep & ~low;
    holes_at.count<kGroups>(hole);
    src_at.count<kGroups>(src);
    const int4 sum = warps_before(holes_at.warp_total(), src_at.warp_total(), sh.warp_sum);
    holes_at.base = sum.x;
    src_at.base = sum.y;
    round_holes = sum.z;
    round_src = sum.w;
  };
  if (C > 1) {
    int ties = tie_base, n_hole = 0, n_src = 0;
#pragma unroll 1
    for (int round = 0; round < rounds; ++round) {
      if (rounds > 1) load_keys(round);
      rank_round(ties);
      n_hole += round_holes;
      n_src += round_src;
    }
    if (tid == 0) {
      sh.total[0] = n_hole;
      sh.total[1] = n_src;
    }
    cluster_sync();
    const int4 x = before(sh.total);
    hole_base = x.x;
    src_base = x.y;
    hole_all = x.z;
  }
  {
    int ties = tie_base, n_hole = hole_base, n_src = src_base;
#pragma unroll 1
    for (int round = 0; round < rounds; ++round) {
      if (rounds > 1) load_keys(round);
      if (rounds > 1 || C == 1) rank_round(ties);  // else the ranks are still there
#pragma unroll
      for (int q = 0; q < kGroups; ++q) {
        int hr = n_hole + holes_at.group(q), sr = n_src + src_at.group(q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * q + e;
          if (hole >> i & 1u) holes[hr++] = static_cast<int32_t>(row_of(i));
          if (src >> i & 1u) sources[sr++] = static_cast<int32_t>(row_of(i));
        }
      }
      n_hole += round_holes;
      n_src += round_src;
      if (C == 1) hole_all = n_hole;
    }
  }
  sync_all();  // the lists are complete
  if (C > 1 ? sh.bad != 0 : __any_sync(0xffffffffu, lane < T >> 5 && sh.found[lane])) {
    leave();
    return;
  }
  for (int k = rank * T + tid; k < hole_all; k += C * T) {
    const int d = holes[k], q = sources[k];
    kept[d] = q;
    if (C == 1 && w_out) w_out[d] = w[q];
    if (C == 1 && p_out) p_out[d] = pos ? pos[q] : q;
  }
  if (C > 1) {
    // All CTAs of the cluster together: the rows below the budget are few CTAs' own.
    cluster_sync();
    for (int r = rank * T + tid; r < n; r += 2 * C * T) {
      const int r2 = r + C * T < n ? r + C * T : r;
      const int q = kept[r], q2 = kept[r2];
      const float x = w[q], x2 = w[q2];
      const int32_t y = pos ? pos[q] : q, y2 = pos ? pos[q2] : q2;
      if (w_out) {
        w_out[r] = x;
        w_out[r2] = x2;
      }
      if (p_out) {
        p_out[r] = y;
        p_out[r2] = y2;
      }
    }
  }
  put_aside(hole_all);
}

#pragma nv_diagnostic pop

// The rows of 8-bit caches where moves can be as many as blocks: a warp has one
// block's keys or values. Else by list entries. (128 heads to 3001 rows of e4m3, 188
// blocks: 40 moves 37.4 us by entries and 36.3 by blocks, 100 moves 46.5 and 47.1,
// 188 57.2 and 54.8, 500 75.1 and 68.3.)
template <int KIND, int D>
__global__ void __launch_bounds__(32 * kMoveWarps, 4) cache_move_kernel(const EvictArgs a, int32_t chunks, int64_t items) {
  __shared__ MoveSlot all_slots[kMoveWarps][32];
  MoveSlot* const slots = all_slots[threadIdx.x >> 5];
  int64_t item = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
  if (item >= items) return;
  const int lane = threadIdx.x & 31;
  const int kv = cache_8bit(KIND) ? static_cast<int>(item & 1) : 0;
  if (cache_8bit(KIND)) item >>= 1;
  const int64_t pair = item / chunks;
  const int chunk = static_cast<int>(item % chunks);
  const int h = static_cast<int>(pair % a.c.Hkv), b = static_cast<int>(pair / a.c.Hkv);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int m = a.counts[pair];
  if (!cache_8bit(KIND) || !a.by_block) {
    if (chunk * move_entries(KIND) < m) move_entries_of<KIND, D>(a, pair, b, h, chunk, kv, m, slots);
    return;
  }
  const int lo = chunk * a.c.scale_block;
  const int hi = a.budget - lo > a.c.scale_block ? lo + a.c.scale_block : a.budget;
  const int32_t* kept = a.kept + pair * a.budget;
  const int src0 = lo + lane < hi ? kept[lo + lane] : lo + lane;  // asked for together with m
  bool moved = src0 != lo + lane;
  for (int r = lo + lane + 32; r < hi; r += 32) moved = moved || kept[r] != r;
  if (m > 0 && __any_sync(0xffffffffu, moved)) move_block<KIND, D>(a, kv, b, h, pair, lo, src0, slots);
}

struct EvictPlan {
  CacheView c;
  int64_t list;    // most moves of a (sequence, kv head)
  int32_t chunks;  // warps of `move` for each of them (and for keys and values, in 8 bits)
  bool by_block;   // a chunk is a scale block, else list entries
  size_t bytes;
};

pa_status plan_evict(const pa_block_cache_desc* d, bool paged, int64_t budget, EvictPlan* p) {
  *p = EvictPlan{};
  PA_TRY(check_cache(d, {paged, true, false}, &p->c, "cache evict"));
  if (budget < 1 || budget > 0x7fffffffLL - 1024) return fail(PA_ERR_INVALID, "cache evict: budget must be in [1, 2^31)");
  const size_t pairs = static_cast<size_t>(p->c.B) * p->c.Hkv;
  const int64_t over = p->c.max_len > budget ? p->c.max_len - budget : 0;
  p->list = over < budget ? over : budget;
  p->bytes = pairs * (3 + 2 * static_cast<size_t>(p->list)) * sizeof(int32_t);
  int64_t chunks = (p->list + move_entries(p->c.kind) - 1) / move_entries(p->c.kind);
  if (cache_8bit(p->c.kind)) {
    const int64_t blocks = (budget + p->c.scale_block - 1) / p->c.scale_block;
    p->by_block = p->list >= blocks;
    if (p->by_block) chunks = blocks;
  }
  p->chunks = static_cast<int32_t>(chunks);
  if (pairs * kMaxCluster > 0x7fffffffu || static_cast<int64_t>(pairs) * 2 * chunks / kMoveWarps >= 0x7fffffffLL)
    return fail(PA_ERR_UNSUPPORTED, "cache evict: grid too large");
  return PA_OK;
}

// A CTA per (sequence, kv head), or a cluster of 2, 4 or 8 while each CTA then has
// an SM and 2048 rows (128 heads of 8191 rows: 44.0 us alone, 49.0 in pairs);
// threads for eight rows each, sixteen where 1024 threads of eight would need a
// second round. Where max_seq_len lets no sequence be more than kFewRows over the
// budget, the CTA carries the rows over itself (one row of 2049 in 512 heads: 14.4 us,
// with a second launch 16.9).
template <int KIND, int D>
pa_status launch_evict(EvictArgs a, int32_t chunks, cudaStream_t st) {
  const int64_t pairs = static_cast<int64_t>(a.c.B) * a.c.Hkv;
  int cluster = 1;
  while (cluster < kMaxCluster && pairs * cluster * 2 <= sm_count() && a.c.max_len / (2 * cluster) >= 2048) cluster *= 2;
  a.cluster = cluster;
  const int64_t share = (static_cast<int64_t>(a.c.max_len) + cluster - 1) / cluster;
  const int keys = share > 8 * kMaxThreads ? 16 : 8;
  int64_t threads = ((share + keys - 1) / keys + 31) / 32 * 32;
  threads = threads < kScanThreads ? kScanThreads : threads > kMaxThreads ? kMaxThreads : threads;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(pairs * cluster));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = sizeof(EvictShared);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  if (a.c.max_len - a.budget <= kFewRows && a.list > 0 && cluster == 1 && share <= threads * 8 && threads <= 320) {
    PA_CUDA(cudaLaunchKernelEx(&cfg, cache_select_kernel<8, 320, 4, KIND, D>, a));
    return PA_OK;
  }
  PA_CUDA(cudaLaunchKernelEx(&cfg, keys == 16       ? cache_select_kernel<16, kMaxThreads, 1, -1, 0>
                                   : threads <= 320 ? cache_select_kernel<8, 320, 4, -1, 0>
                                                    : cache_select_kernel<8, kMaxThreads, 1, -1, 0>, a));
  if (a.list == 0) return PA_OK;
  const int64_t items = pairs * chunks * (cache_8bit(KIND) ? 2 : 1);
  // Starts while `select` ends; waits for its memory.
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(static_cast<unsigned>((items + kMoveWarps - 1) / kMoveWarps));
  cfg.blockDim = dim3(32 * kMoveWarps);
  cfg.dynamicSmemBytes = 0;
  PA_CUDA(cudaLaunchKernelEx(&cfg, cache_move_kernel<KIND, D>, a, chunks, items));
  return PA_OK;
}

template <int D>
pa_status launch_evict_kind(const EvictArgs& a, int32_t chunks, cudaStream_t st) {
  switch (a.c.kind) {
    case kCacheF16:
    case kCacheBF16: return launch_evict<kCacheF16, D>(a, chunks, st);  // rows are copied as bits
    case kCacheE4M3: return launch_evict<kCacheE4M3, D>(a, chunks, st);
    default: return launch_evict<kCacheI8, D>(a, chunks, st);
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
  if (seq_lens_out == next_positions) return fail(PA_ERR_INVALID, "cache evict: seq_lens_out must not be next_positions");
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
  a.list = static_cast<int32_t>(p.list);
  a.by_block = p.by_block;
  a.vec = ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(positions) |
            reinterpret_cast<uintptr_t>(weights_out) | reinterpret_cast<uintptr_t>(positions_out)) & 15) == 0 &&
          p.c.row_head % 4 == 0 && p.c.row_seq % 4 == 0;
  a.vec_kept = (reinterpret_cast<uintptr_t>(kept) & 15) == 0 && budget % 4 == 0;
  void* own = nullptr;
  if (!workspace) PA_TRY(scratch_alloc(&own, p.bytes, st));
  const size_t pairs = static_cast<size_t>(p.c.B) * p.c.Hkv;
  a.cut_scale = static_cast<float*>(workspace ? workspace : own);
  a.counts = reinterpret_cast<int32_t*>(a.cut_scale + pairs * 2);
  a.holes = a.counts + pairs;
  a.sources = a.holes + pairs * p.list;
  pa_status rc = p.c.D == 128 ? launch_evict_kind<128>(a, p.chunks, st) : launch_evict_kind<64>(a, p.chunks, st);
  scratch_free(own, st);
  return rc;
}
