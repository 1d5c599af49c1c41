// What the kernels that decode against a paged KV cache share (paged_decode.cu: rows in 16 and 32 bits, paged_4bit.cu: rows in 4
// bits): the list of stages and a warp's share of it, a warp's ring of copies, what a block does around its warps' walks, and the
// fold of the parts that the shares leave. paged_decode.cu tells why the work is dealt so.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "mma16.cuh"
#include "paged.cuh"
#include "tc_common.cuh"

namespace rab {

namespace {

using tcgen::ex2;
using tcgen::kLn2;
using tcgen::kLog2e;

struct PagedArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;  // or NULL
  const int* table;
  long long table_stride;
  const int* lens;
  const int* shared_pages;
  int shared_len;  // rows in shared pages that are read once for the batch
  int listed_len;  // or rows that a sequence which has all of them reads from shared_pages instead of its table
  int num_pages, max_pages, shift;
  int B, H, kvH;
  int G;   // heads of a KV head, at most
  int HB;  // units of a KV head and a sequence
  int RB;  // units of a KV head on the shared pages (0: not by this kernel)
  int rs;  // rows of a part in the workspace
  float scale_log2;
  int2* unit_parts;  // first share that has a part of a unit, and how many do
  float2* part_ml;   // (m in log2 units, l) of rs rows, a part after the other
  float* part_o;
  // shared pages by the tensor-core kernel (step_tc.cu; RB is 0 then): its parts, see SharedPrefix
  SharedPlan shared;
  float2* shared_ml;  // NULL: not by it
  float* shared_o;
  int* status;
  unsigned long long wait_ns;
  int shares;   // that the stages are dealt in
  int missing;  // (test hook: bytes that every stage waits for in vain; 0: none; -1: no warp does anything)
};

// Keys [start, end) of a sequence that its own table holds: behind the shared pages if it has all of them.
__device__ inline void own_keys(const PagedArgs& a, int b, int* start, int* end) {
  const long long len = min(static_cast<long long>(a.lens[b]), static_cast<long long>(a.max_pages) << a.shift);
  *end = len > 0 ? static_cast<int>(min(len, 0x7fffffffll)) : 0;
  *start = a.shared_len > 0 && *end >= a.shared_len ? a.shared_len : 0;
}
template <int SR>
__device__ inline int own_stages(const PagedArgs& a, int b) {
  int start, end;
  own_keys(a, b, &start, &end);
  return static_cast<int>((static_cast<long long>(end) - start + SR - 1) / SR);
}

// A place in the list of stages.
template <int SR>
struct Walk {
  int uid;         // number of the unit; units on the shared pages come first
  int b, kvh, hb;  // b = -1: on the shared pages
  int st, n;       // stage of the unit and how many it has
  int start, end;  // its keys
  int listed;      // so many pages from the list of shared pages
  __device__ inline int shared_stages(const PagedArgs& a) const { return (a.shared_len + SR - 1) / SR; }
  __device__ inline void on_shared(const PagedArgs& a) {
    b = -1;
    start = 0;
    end = a.shared_len;
    listed = a.shared_len >> a.shift;
    n = shared_stages(a);
  }
  __device__ inline void on_sequence(const PagedArgs& a, int seq) {
    b = seq;
    own_keys(a, b, &start, &end);
    listed = end >= a.listed_len ? a.listed_len >> a.shift : 0;
    n = static_cast<int>((static_cast<long long>(end) - start + SR - 1) / SR);
  }
  __device__ inline void number(const PagedArgs& a) { uid = b < 0 ? kvh * a.RB + hb : a.kvH * a.RB + (b * a.kvH + kvh) * a.HB + hb; }
  __device__ inline int left() const { return end - start - st * SR; }  // keys from this stage on
  // On to the next stage; there has to be one.
  __device__ inline void next(const PagedArgs& a) {
    if (++st < n) return;
    st = 0;
    if (++hb == (b < 0 ? a.RB : a.HB)) {
      hb = 0;
      if (++kvh == a.kvH) {
        kvh = 0;
        int seq = b;
        do on_sequence(a, ++seq);
        while (n == 0 && seq + 1 < a.B);
      }
    }
    number(a);
  }
};

// Room of find_share.
template <int kWarps>
struct ScanRoom {
  long long sums[kWarps];
  long long in_seq[kWarps];
  int seq[kWarps];
};

// Sum over the block of a thread's v, and the sum over the threads before it.
template <int kWarps>
__device__ inline long long block_scan(long long v, long long* total, ScanRoom<kWarps>* room) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = v;
#pragma unroll
  for (int i = 1; i < 32; i *= 2) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, i);
    if (lane >= i) incl += o;
  }
  __syncthreads();
  if (lane == 31) room->sums[warp] = incl;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += room->sums[w];
    all += room->sums[w];
  }
  *total = all;
  return before + incl - v;
}

// The warp's share: its first place, and how many stages (0: none); *per: stages of a whole share. Every thread of the block calls.
template <int SR, int kWarps>
__device__ inline int find_share(const PagedArgs& a, int warp, Walk<SR>* w, int* per, ScanRoom<kWarps>* room) {
  constexpr int kThreads = 32 * kWarps;
  const int units = a.kvH * a.HB;
  long long shared_total = 0;
  if (a.RB > 0) shared_total = static_cast<long long>(a.kvH) * a.RB * w->shared_stages(a);
  // the first chunk of sequences stays at hand
  const int mine = static_cast<int>(threadIdx.x) < a.B ? own_stages<SR>(a, threadIdx.x) : 0;
  long long sum = mine, total;
  for (int b = static_cast<int>(threadIdx.x) + kThreads; b < a.B; b += kThreads) sum += own_stages<SR>(a, b);
  const long long before = block_scan<kWarps>(sum, &total, room);
  const long long all = shared_total + total * units, shares = static_cast<long long>(gridDim.x) * kWarps;
  const long long share = max(1ll, (all + shares - 1) / shares);
  *per = static_cast<int>(share);
  const long long first_of_block = share * blockIdx.x * kWarps, end_of_block = min(first_of_block + share * kWarps, all);
  if (end_of_block > shared_total) {
    long long base = shared_total;
    for (int b0 = 0; b0 < a.B && base < end_of_block; b0 += kThreads) {
      const int b = b0 + static_cast<int>(threadIdx.x);
      long long n = mine, chunk = total, ahead = before;  // (of the only chunk)
      if (a.B > kThreads) {
        if (b0 > 0) n = b < a.B ? own_stages<SR>(a, b) : 0;
        ahead = block_scan<kWarps>(n, &chunk, room);
      }
      const long long at = base + ahead * units;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const long long first = first_of_block + share * i;
        if (first >= at && first < at + n * units) {
          room->seq[i] = b;
          room->in_seq[i] = first - at;
        }
      }
      base += chunk * units;
    }
  }
  __syncthreads();
  const long long first = first_of_block + share * warp, stages = min(share, all - first);
  if (stages <= 0) return 0;
  if (first < shared_total) {
    w->on_shared(a);
    const int u = static_cast<int>(first / w->n);
    w->st = static_cast<int>(first - static_cast<long long>(u) * w->n);
    w->kvh = u / a.RB;
    w->hb = u % a.RB;
  } else {
    w->on_sequence(a, room->seq[warp]);
    const long long in_seq = room->in_seq[warp];
    const int u = static_cast<int>(in_seq / w->n);
    w->st = static_cast<int>(in_seq - static_cast<long long>(u) * w->n);
    w->kvh = u / a.HB;
    w->hb = u % a.HB;
  }
  w->number(a);
  return static_cast<int>(stages);
}

// What a warp has to know of a stage when its copy has landed.
struct StageInfo {
  int b, kvh, hb, uid;
  int keys;        // of the stage
  unsigned pages;  // bit i: keys 16 i and on are there
  int first;       // of the warp's part of the unit
  int last;        // the same; 2: and the part is the result, the unit being whole and no shared pages ahead of it
};

// Query row r of a unit: sequence and head; false where the unit has no such row.
template <int RU>
__device__ inline bool unit_row(const PagedArgs& a, const StageInfo& u, int r, int* b, int* h) {
  const int i = u.hb * RU + r, g = u.b < 0 ? i % a.G : i;
  *b = u.b < 0 ? i / a.G : u.b;
  *h = u.kvh + a.kvH * g;
  return *b < a.B && *h < a.H;
}

// What the kernels are built with and the host sizes the workspace by: keys of a stage, warps of a block, and rows of a unit in 16
// bits (fp32: see fp32_rows).
constexpr int stage_keys(bool f32, int D) { return f32 ? (D == 32 ? 32 : D == 64 ? 16 : 8) : D <= 64 ? 32 : 16; }
constexpr int block_warps(bool f32, int D) { return D == 256 ? 2 : D == 32 && !f32 ? 8 : 4; }  // (64 bytes a row: more, for its instructions)
constexpr int kMmaRows = 16;

// Shared memory of a block of either kernel: the rings of its warps, a stage being SR rows of K and then of V. 16 bits: a tensor's
// kBoxes boxes of 128 bytes of every row, by tensor maps, 16-byte piece c of a row's box at c ^ (row & 7) (rows of 64 bytes: one
// box of those, c ^ (row / 2 & 3)). fp32: whole rows, one
// after the other as in the page, by plain bulk copies (boxes of 8 rows and 128 bytes kept TMA busy: 16384 rows of D128 67 us).
// The shorter a row, the more of them a stage and the more warps, for the instructions around a stage: us a pass, four sequences of
// 131072 to 262144 rows (H32/kvH8 fp16), head_dim 64 in stages of 16 / 32 rows 324 / 254; head_dim 32 in stages of 16 rows that fill
// 128 bytes each, four / eight warps 294 / 178, of 32 rows of 64 bytes, eight warps, 138.
template <typename T, int D, int kRows_, int kExtraBytes>
struct PagedBlock {
  static constexpr bool kBulk = sizeof(T) == 4;
  static constexpr int SR = stage_keys(kBulk, D), RU = kRows_;
  static constexpr int kWarps = block_warps(kBulk, D), kThreads = kWarps * 32;
  static constexpr int kBoxes = kBulk || D <= 64 ? 1 : D / 64;
  static constexpr int kBoxBytes = D == 32 && !kBulk ? 64 : 128;
  static constexpr int kRowBytes = kBulk ? D * 4 : kBoxes * kBoxBytes;  // in shared memory
  static constexpr int kTileBytes = SR * kRowBytes;               // per tensor
  static constexpr int kStages = 96 * 1024 / kWarps / (2 * kTileBytes);
  static constexpr int kRingBytes = 2 * kStages * kTileBytes;  // of a warp
  static constexpr int kOffExtra = kWarps * kRingBytes;        // fp32: every warp's weights and factors
  static constexpr int kOffInfo = kOffExtra + kWarps * kExtraBytes;
  static constexpr int kOffBar = kOffInfo + kWarps * kStages * static_cast<int>(sizeof(StageInfo));
  static constexpr int kOffRoom = kOffBar + kWarps * kStages * 8;
  static constexpr int kOffFlag = kOffRoom + static_cast<int>(sizeof(ScanRoom<kWarps>));
  static constexpr int kSmemBytes = kOffFlag + 8;
  static_assert(kTileBytes % 1024 == 0 && kStages >= 3, "the ring");
  static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two blocks to an SM");
};

// A warp's ring: copies run kStages - 1 stages ahead of what it computes.
template <typename C>
struct Ring {
  const PagedArgs& a;
  const CUtensorMap *map_k, *map_v;
  unsigned tiles, full;  // shared memory: the ring, its barriers
  StageInfo* info;
  volatile int* gave_up;
  Walk<C::SR> w;         // the next stage to copy
  int total, per, next = 0, first_st;
  int head[C::kStages];  // this lane's page of the next stages, as far as they are looked up (see look_up)

  // A lane's copies: a piece of the stage's rows (two where a stage takes 32 and a page has 16), a box of one tensor.
  static_assert(C::SR <= 32 && 2 * C::kBoxes * ((C::SR + 15) / 16) <= 32, "a copy a lane");
  __device__ inline bool halved() const { return C::SR == 32 && a.shift == 4; }
  __device__ inline int rows() const { return halved() ? 16 : C::SR; }
  // The page of this lane's piece, as the head its rows are in the tensor map; -1 where there is none.
  __device__ inline int look_up(const Walk<C::SR>& w) const {
    const int first = halved() ? static_cast<int>(threadIdx.x & 1) * 16 : 0;  // row of the piece
    if (first >= w.left()) return -1;
    const int at = (w.start + w.st * C::SR + first) >> a.shift;
    if (at >= w.listed && (w.b < 0 || at >= a.max_pages)) return -1;
    const int page = at < w.listed ? a.shared_pages[at] : a.table[w.b * a.table_stride + at];
    return page >= 0 && page < a.num_pages ? page * a.kvH + w.kvh : -1;
  }
  // Looks the first stages up together, so that their copies do not wait for one another's page numbers, and copies them.
  __device__ inline void begin() {
    first_st = w.st;
    Walk<C::SR> ahead = w;
#pragma unroll
    for (int s = 0; s < C::kStages; ++s) {
      head[s] = s < total ? look_up(ahead) : -1;
      if (s + 1 < total) ahead.next(a);
    }
#pragma unroll
    for (int s = 0; s < C::kStages; ++s) copy(s, head[s]);
    if (next < total) head[0] = look_up(w);
  }
  // Copies the next stage, if there is one, to a place that is free, and looks the one behind it up.
  __device__ inline void copy_next(int slot) {
    if (next >= total) return;
    copy(slot, head[0]);
    if (next < total) head[0] = look_up(w);
  }
  __device__ inline void copy(int slot, int head) {
    if (next >= total) return;
    const int lane = threadIdx.x & 31, pieces = halved() ? 2 : 1, at = halved() ? lane >> 1 : lane;
    const int first = halved() ? (lane & 1) * 16 : 0, box = at % C::kBoxes, tensor = at / C::kBoxes;
    if (w.st == 0) {
      first_st = 0;
      // the warp with a unit's first stage says which shares have parts of it: its own and those that the rest reaches into
      const int here = min(w.n, total - next);
      if (lane == 0)
        a.unit_parts[w.uid] = make_int2(static_cast<int>(blockIdx.x * C::kWarps + (threadIdx.x >> 5)), 1 + (w.n - here + per - 1) / per);
    }
    const int row = (w.start + w.st * C::SR + first) & ((1 << a.shift) - 1);
    const unsigned there = __ballot_sync(0xffffffffu, head >= 0 && lane < pieces);
    if (lane == 0) {
      StageInfo i;
      i.b = w.b, i.kvh = w.kvh, i.hb = w.hb, i.uid = w.uid;
      i.keys = min(C::SR, w.left());
      i.pages = there;
      if (C::SR > 16 && pieces == 1) i.pages |= there << 1;  // (a page of 32 keys and more)
      const bool ends = w.st == w.n - 1;
      i.first = w.st == first_st;
      i.last = ends && first_st == 0 && w.b >= 0 && w.start == 0 ? 2 : ends || next == total - 1;
      info[slot] = i;
      tcgen::mbar_expect_tx(full + 8 * slot, 2 * C::kRowBytes * rows() * __popc(there) + a.missing);
    }
    __syncwarp();
    if constexpr (C::kBulk) {
      if (tensor < 2 && head >= 0)
        tcgen::bulk_load(tiles + (2 * slot + tensor) * C::kTileBytes + first * C::kRowBytes,
                         static_cast<const unsigned char*>(tensor == 0 ? a.k : a.v) +
                             ((static_cast<size_t>(head) << a.shift) + row) * C::kRowBytes,
                         C::kRowBytes * rows(), full + 8 * slot);
    } else if (tensor < 2 && head >= 0) {
      tcgen::tma_load_3d(tiles + (2 * slot + tensor) * C::kTileBytes + (box * C::SR + first) * C::kBoxBytes,
                         tensor == 0 ? map_k : map_v, full + 8 * slot, box * 64, row, head);
    }
    if (++next < total) w.next(a);
  }
  // Waits for stage s; false: the warp gives up.
  __device__ inline bool wait(int s) {
    return __all_sync(0xffffffffu, tcgen::mbar_wait(full + 8 * (s % C::kStages), (s / C::kStages) & 1, gave_up, a.status, 3, s,
                                                    a.wait_ns)) != 0;
  }
};

// What a block does around its warps' walks; compute(ring, warp) is a warp's.
template <typename C, typename Compute>
__device__ inline void paged_block(const PagedArgs& a, const CUtensorMap* map_k, const CUtensorMap* map_v, unsigned char* smem,
                                   Compute compute) {
  const unsigned base = tcgen::smem_u32(smem);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  volatile int* const gave_up = reinterpret_cast<volatile int*>(smem + C::kOffFlag);
  let_next_start();
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kWarps * C::kStages; ++s) tcgen::mbar_init(base + C::kOffBar + 8 * s, 1);
    *gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if constexpr (!C::kBulk) {
      tcgen::prefetch_map(map_k);
      tcgen::prefetch_map(map_v);
    }
  }
  // Behind the kernel of the shared pages, whose blocks let this one begin when all that came before them has completed,
  // nothing waits for that kernel itself but the end: the fold, which waits for this grid, then finds both kernels' parts.
  // A grid that begins early is promised nothing about memory, so fences stand for the wait's other half: that kernel's threads
  // have one between their wait and the signal, these have one behind it, and one more for the copies, which read what plain
  // stores wrote (an append's rows). us a pass in a graph, 256 sequences behind 16384 rows and 32 behind 32768 (H32/kvH8 D128 bf16): so
  // 146.7 and 54.2, waiting here 154.4 and 54.5, without the fences 146.5 and 53.9.
  if (a.shared_ml == nullptr) {
    wait_for_previous();
  } else {
    __threadfence();
    asm volatile("fence.proxy.async.global;" ::: "memory");
  }
  Ring<C> ring{a, map_k, map_v, base + warp * C::kRingBytes, base + C::kOffBar + warp * C::kStages * 8,
               reinterpret_cast<StageInfo*>(smem + C::kOffInfo) + warp * C::kStages, gave_up};
  ring.total = find_share<C::SR, C::kWarps>(a, warp, &ring.w, &ring.per, reinterpret_cast<ScanRoom<C::kWarps>*>(smem + C::kOffRoom));
  // (behind a launch that gave up nothing is computed; the fold writes nothing then either)
  if (ring.total > 0 && a.missing >= 0 && __shfl_sync(0xffffffffu, *reinterpret_cast<volatile int*>(a.status), 0) == 0) {
    ring.begin();
    compute(ring, warp);
  }
  __syncthreads();
  if (*gave_up) {  // give copies in flight time to land
    const unsigned long long t0 = tcgen::global_ns();
    while (tcgen::global_ns() - t0 < 1000000ull) __nanosleep(1000);
  }
  if (a.shared_ml != nullptr) wait_for_previous();
}

// ---- fold ---------------------------------------------------------------------------

struct Acc8 {  // eight columns of a row
  float4 lo, hi;
};
__device__ inline Acc8 scaled(float f, const Acc8& a) {
  return {make_float4(f * a.lo.x, f * a.lo.y, f * a.lo.z, f * a.lo.w), make_float4(f * a.hi.x, f * a.hi.y, f * a.hi.z, f * a.hi.w)};
}
__device__ inline void add_scaled(Acc8& s, float f, const Acc8& a) {
  s.lo.x = fmaf(f, a.lo.x, s.lo.x), s.lo.y = fmaf(f, a.lo.y, s.lo.y), s.lo.z = fmaf(f, a.lo.z, s.lo.z), s.lo.w = fmaf(f, a.lo.w, s.lo.w);
  s.hi.x = fmaf(f, a.hi.x, s.hi.x), s.hi.y = fmaf(f, a.hi.y, s.hi.y), s.hi.z = fmaf(f, a.hi.z, s.hi.z), s.hi.w = fmaf(f, a.hi.w, s.hi.w);
}
__device__ inline float4 shfl4(float4 v, int d) {
  return make_float4(__shfl_xor_sync(0xffffffffu, v.x, d), __shfl_xor_sync(0xffffffffu, v.y, d), __shfl_xor_sync(0xffffffffu, v.z, d),
                     __shfl_xor_sync(0xffffffffu, v.w, d));
}

// Parts of the rows that no warp finished, and rows without keys. A row's kCols columns have kCols / 8 threads, eight columns each,
// times kSlices, which take every kSlices-th part; a thread asks for eight parts at a time, or, where there are many rows, for four.
template <typename T, int D, int RU, int kFoldThreads, int kSlices, int kCols>
__global__ void __launch_bounds__(kFoldThreads) paged_fold_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int kVec = kCols / 8, kRowsPer = kFoldThreads / kVec / kSlices, kBatch = kSlices >= 8 ? 8 : 4;
  // slices that sit in one warp meet by shuffles, the others (kGroups of a row) through shared memory
  constexpr int kInWarp = kSlices < 32 / kVec ? kSlices : 32 / kVec, kGroups = kSlices / kInWarp;
  __shared__ Acc8 acc_of[kGroups > 1 ? kFoldThreads / kInWarp : 1];
  __shared__ float m_of[kGroups > 1 ? kFoldThreads / kVec / kInWarp : 1], l_of[kGroups > 1 ? kFoldThreads / kVec / kInWarp : 1];
  let_next_start();
  const int col = (static_cast<int>(blockIdx.y) * kVec + threadIdx.x % kVec) * 8, lane_row = threadIdx.x / kVec, slice = lane_row % kSlices;
  const int row = static_cast<int>(blockIdx.x) * kRowsPer + lane_row / kSlices;
  const bool mine = row < a.B * a.H;
  const int b = mine ? row / a.H : 0, h = mine ? row - b * a.H : 0, kvh = h % a.kvH, g = h / a.kvH;
  const int own_uid = a.kvH * a.RB + (b * a.kvH + kvh) * a.HB + g / RU;
  const int of_all = b * a.G + g, shared_uid = a.RB > 0 ? kvh * a.RB + of_all / RU : own_uid;
  // the row's first part of the shared pages, and how far the next one is
  int pre_n = 0;
  long long pre_lo = 0, pre_step = a.rs;
  const float2* pre_ml = a.part_ml;
  const float* pre_o = a.part_o;
  if (a.shared_ml) {
    const SharedPlan& s = a.shared;
    const int tile = s.pack > 1 ? g / s.pack : b / 128 * a.G + g, at = s.pack > 1 ? g % s.pack * a.B + b : b % 128;
    pre_step = s.tiles_per_block * 128;
    pre_lo = (static_cast<long long>(kvh) * s.blocks + tile / s.tiles_per_block) * s.shares * pre_step + tile % s.tiles_per_block * 128 + at;
    pre_n = s.shares;
    pre_ml = a.shared_ml;
    pre_o = a.shared_o;
  }
  wait_for_previous();
  bool lost = *reinterpret_cast<const volatile int*>(a.status) != 0;  // some wait ran out: the rows stay as they are
  const int2 own = a.unit_parts[own_uid], pre = a.unit_parts[shared_uid];
  int start = 0, end = 0;
  if (mine) own_keys(a, b, &start, &end);
  // So they do where no warp of this call has said which parts there are: the word was set when the warps looked at it, and another
  // thread of the host has read and cleared it since. What the workspace holds in that place may be anything.
  auto said = [&](const int2& p) { return p.x >= 0 && p.y > 0 && p.y <= a.shares - p.x; };
  if ((end > start && !said(own)) || (start > 0 && !a.shared_ml && !said(pre))) lost = true;
  const int own_n = end > start ? own.y : 0;
  const long long own_lo = (static_cast<long long>(own.x) + own_uid) * a.rs + g % RU;
  if (!a.shared_ml) {
    pre_lo = (static_cast<long long>(pre.x) + shared_uid) * a.rs + of_all % RU;
    pre_n = pre.y;
  }
  if (start == 0) pre_n = 0;
  const bool done = lost || (own_n == 1 && start == 0);  // by the warp that had the unit
  const int parts = mine && !done ? own_n + pre_n : 0;
  float m_all = -INFINITY, l_all = 0.f;
  Acc8 acc = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int i0 = slice; i0 < parts; i0 += kSlices * kBatch) {
    float2 ml[kBatch];
    Acc8 o[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kSlices;
      ml[j] = make_float2(-INFINITY, 0.f);
      if (i < parts) {
        const bool is_pre = i < pre_n;
        const long long at = is_pre ? pre_lo + i * pre_step : own_lo + static_cast<long long>(i - pre_n) * a.rs;
        ml[j] = (is_pre ? pre_ml : a.part_ml)[at];
        const float4* const src = reinterpret_cast<const float4*>((is_pre ? pre_o : a.part_o) + at * D + col);
        o[j].lo = src[0];
        o[j].hi = src[1];
      }
    }
    float m_new = m_all;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) m_new = fmaxf(m_new, ml[j].x);
    const float f_old = m_all == -INFINITY ? 1.f : ex2(m_all - m_new);
    l_all *= f_old;
    acc = scaled(f_old, acc);
    m_all = m_new;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (ml[j].y == 0.f) continue;  // saw nothing, and may have left no O
      const float f = ml[j].x > -INFINITY ? ex2(ml[j].x - m_all) : 1.f;
      l_all += f * ml[j].y;
      add_scaled(acc, f, o[j]);
    }
  }
  // the slices of a row: the largest m of all, then plain sums
  T* const out = static_cast<T*>(a.out) + static_cast<size_t>(row) * D;
  if constexpr (kSlices > 1) {
    float m_row = m_all;
#pragma unroll
    for (int d = kVec; d < kVec * kInWarp; d *= 2) m_row = fmaxf(m_row, __shfl_xor_sync(0xffffffffu, m_row, d));
    const int group = lane_row / kInWarp, first_group = lane_row / kSlices * kGroups;  // (a row's groups lie one after the other)
    if constexpr (kGroups > 1) {
      if (threadIdx.x % (kVec * kInWarp) == 0) m_of[group] = m_row;
      __syncthreads();
#pragma unroll 8
      for (int k = 0; k < kGroups; ++k) m_row = fmaxf(m_row, m_of[first_group + k]);
    }
    const float f = m_all > -INFINITY ? ex2(m_all - m_row) : 1.f;
    m_all = m_row;
    l_all *= f;
    acc = scaled(f, acc);
#pragma unroll
    for (int d = kVec; d < kVec * kInWarp; d *= 2) {
      l_all += __shfl_xor_sync(0xffffffffu, l_all, d);
      add_scaled(acc, 1.f, {shfl4(acc.lo, d), shfl4(acc.hi, d)});
    }
    if constexpr (kGroups > 1) {
      const int at = threadIdx.x % kVec;
      if (slice % kInWarp == 0) {
        acc_of[group * kVec + at] = acc;
        if (at == 0) l_of[group] = l_all;
      }
      __syncthreads();
      if (!mine || done) return;
      l_all = 0.f;
#pragma unroll 8
      for (int k = 0; k < kGroups; ++k) l_all += l_of[first_group + k];
      const bool any = l_all != 0.f;  // (NaN counts)
      const float inv = any ? 1.f / l_all : 0.f;
      const int mine_of = threadIdx.x % (kVec * kSlices);  // the row's threads take a column at a time
      for (int c = mine_of; c < kCols; c += kVec * kSlices) {
        float sum = 0.f;
#pragma unroll 8
        for (int k = 0; k < kGroups; ++k) sum += reinterpret_cast<const float*>(acc_of)[(first_group + k) * kCols + c];
        out[static_cast<int>(blockIdx.y) * kCols + c] = static_cast<T>(any ? sum * inv : 0.f);
      }
      if (a.lse && blockIdx.y == 0 && mine_of == 0) a.lse[row] = l_all > 0.f ? m_all * kLn2 + logf(l_all) : any ? l_all : -INFINITY;
      return;
    }
  }
  if (!mine || done || slice != 0) return;
  const bool any = l_all != 0.f;  // (NaN counts)
  acc = any ? scaled(1.f / l_all, acc) : Acc8{make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(out + col)[0] = acc.lo;
    reinterpret_cast<float4*>(out + col)[1] = acc.hi;
  } else {
    *reinterpret_cast<uint4*>(out + col) = make_uint4(pack_pair<T>(acc.lo.x, acc.lo.y), pack_pair<T>(acc.lo.z, acc.lo.w),
                                                      pack_pair<T>(acc.hi.x, acc.hi.y), pack_pair<T>(acc.hi.z, acc.hi.w));
  }
  if (a.lse && col == 0) a.lse[row] = l_all > 0.f ? m_all * kLn2 + logf(l_all) : any ? l_all : -INFINITY;
}

// ---- launches ------------------------------------------------------------------------

constexpr int kBlocksPerSm = 2;  // of both kernels

template <auto kern, typename C, typename... Args>
int launch_main(int blocks, cudaStream_t stream, const Args&... args) {
  static std::atomic<unsigned long long> smem_set{0};  // once per device and instantiation
  int dev = 0;
  RAB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !(smem_set.load(std::memory_order_acquire) >> dev & 1ull)) {
    RAB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    if (dev >= 0 && dev < 64) smem_set.fetch_or(1ull << dev, std::memory_order_release);
  }
  RAB_CUDA(launch_overlapped(kern, dim3(static_cast<unsigned>(blocks)), dim3(C::kThreads), C::kSmemBytes, stream, args...));
  return RA_OK;
}

// Threads of the fold that share out a row's parts. With few rows the shares of a whole wave may belong to one of them: then 128
// threads share out a row's parts for 32 columns (8 rows, 262144 keys: 58 us without, 33 with); elsewhere as many as leave the
// threads of all rows room on the SMs at once (one for all / as many: 168 rows of 1531 keys 16.5 / 8.5 us, 1024 rows behind 32768
// shared ones 58.3 / 53.6, fp32, 192 rows of 16384 keys 104 / 87).
template <typename T, int D, int RU>
int launch_fold(const PagedArgs& a, cudaStream_t stream) {
  const long long rows = static_cast<long long>(a.B) * a.H, sms = sm_count();
  auto go = [&](auto threads, auto slices, auto cols) -> int {
    constexpr int kThreads = decltype(threads)::value, kSlices = decltype(slices)::value, kCols = decltype(cols)::value;
    constexpr int kPer = kThreads / (kCols / 8) / kSlices;
    RAB_CUDA(launch_overlapped(paged_fold_kernel<T, D, RU, kThreads, kSlices, kCols>,
                               dim3(static_cast<unsigned>((rows + kPer - 1) / kPer), D / kCols), dim3(kThreads), 0, stream, a));
    return RA_OK;
  };
  using std::integral_constant;
  if (rows * (D / 32) <= 2 * sms) return go(integral_constant<int, 512>(), integral_constant<int, 128>(), integral_constant<int, 32>());
  const long long room = sms * 768 / (rows * (D / 8));
  if (room >= 8) return go(integral_constant<int, 256>(), integral_constant<int, 8>(), integral_constant<int, D>());
  if (room >= 4) return go(integral_constant<int, 256>(), integral_constant<int, 4>(), integral_constant<int, D>());
  if (room >= 2) return go(integral_constant<int, 256>(), integral_constant<int, 2>(), integral_constant<int, D>());
  return go(integral_constant<int, 256>(), integral_constant<int, 1>(), integral_constant<int, D>());
}

}  // namespace
}  // namespace rab
