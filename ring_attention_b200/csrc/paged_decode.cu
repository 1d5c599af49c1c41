// Decode attention (one query row a sequence) against a paged KV cache, sequences of any lengths, which only the device knows;
// and for a batch whose sequences begin with the same pages, those once for all.
//
//   out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(q . k_j / sqrt(D)),  j < lens[b],  KV head h % kv_heads
//
// What bounds it is the cache: every row is read once. The work is cut into units, the up to RU query rows that read the same
// keys: the heads of a KV head and a sequence, behind the shared pages where the sequence has them; and for the shared pages RU
// rows of all sequences. A unit is a list of stages of SR keys, and all units' stages one after the other are dealt in equal
// shares to the warps of one wave, so that lengths do not matter to the balance. A unit that lies in one share is finished
// there; of others every share leaves (O, m, l) in the workspace, and a second kernel folds them.
//
// A warp works alone: it walks its share, looks the pages up a stage ahead and copies the rows of a stage with TMA (a piece of a
// page and 128 bytes of its rows a lane, 128-byte swizzle) into a ring of its own, 192 KB for the warps of an SM. Where a unit
// ends and the next one's queries come, and where it waits for a copy, the others of the SM run on. us a pass, four sequences of
// 131072 to 262144 rows (H32/kvH8 D128 fp16) and 256 of 300 to 600: 16-byte cp.async of all threads and a barrier a stage
// 854 and more than 120; a copying warp to four that meet where a unit ends 502 and 103; so 500 and 89. A place of the ring is
// filled again a stage after it was read, so that two stages are on their way and not three: with three the memory
// is the slower for it (528 and 94).
//
// 16-bit caches: both products on mma.sync m16n8k16, the unit's rows as its M rows, as in decode_mma_kernel (decode.cu). fp32:
// plain multiply-adds, 4 to 16 lanes to a key for the scores (see F32Cfg), four columns a lane (head_dim 256: eight) for the sum over V.
//
// Every wait on a barrier is bounded, as in the step kernels: when one runs out the warp records it in the device status word
// and leaves, and the fold leaves every row that it would have written as it is.
//
// Times in this file are of launches one behind the other in a CUDA graph; calls of less than some 15 us wait for the host otherwise.
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

// ---- 16-bit caches ------------------------------------------------------------------

template <typename T, int D>
using MmaBlock = PagedBlock<T, D, kMmaRows, 0>;

template <typename T, int D>
__global__ void __launch_bounds__(MmaBlock<T, D>::kThreads, 2)
    paged_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ PagedArgs a) {
  using C = MmaBlock<T, D>;
  constexpr int SR = C::SR, RU = C::RU, kBoxBytes = C::kBoxBytes, kBoxPieces = kBoxBytes / 16;
  extern __shared__ __align__(1024) unsigned char smem[];
  paged_block<C>(a, &map_k, &map_v, smem, [&](Ring<C>& ring, int warp) {
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2, tq = lane & 3;  // fragment row (and row + 8), column pair
    const int mi = lane >> 3, r8 = lane & 7;
    // a lane's rows of the ldmatrix tiles, and the swizzled offsets of its pieces c = 2 i + (0 or 1) of a box
    const unsigned k_row = ring.tiles + static_cast<unsigned>((mi >> 1) * 8 + r8) * kBoxBytes;
    const unsigned v_row = ring.tiles + static_cast<unsigned>(C::kTileBytes + ((mi & 1) * 8 + r8) * kBoxBytes);
    constexpr int kSteps = kBoxPieces / 2;  // of 16 columns in a box
    const int turn = kBoxBytes == 64 ? r8 >> 1 : r8;
    unsigned k_off[kSteps], v_off[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      k_off[i] = ((2 * i + (mi & 1)) ^ turn) << 4;
      v_off[i] = ((2 * i + (mi >> 1)) ^ turn) << 4;
    }
    unsigned qa[D / 16][4];
    float o[D / 8][4];
    float m_run[2], l_run[2];
    const int total = ring.total;
    for (int s = 0; s < total; ++s) {
      const int slot = s % C::kStages;
      const StageInfo u = ring.info[slot];
      if (u.first) {  // (while the copy is on its way)
        // Q as A fragments: reg0 (row g, k 2tq..), reg1 (row g+8, same k), reg2 / reg3 the same at k+8
        int b0, h0, b1, h1;
        const bool is0 = unit_row<RU>(a, u, g, &b0, &h0), is1 = unit_row<RU>(a, u, g + 8, &b1, &h1);
        const T* const q0 = static_cast<const T*>(a.q) + (is0 ? static_cast<size_t>(b0) * a.H + h0 : 0) * D + 2 * tq;
        const T* const q1 = static_cast<const T*>(a.q) + (is1 ? static_cast<size_t>(b1) * a.H + h1 : 0) * D + 2 * tq;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          qa[ks][0] = is0 ? *reinterpret_cast<const unsigned*>(q0 + ks * 16) : 0u;
          qa[ks][1] = is1 ? *reinterpret_cast<const unsigned*>(q1 + ks * 16) : 0u;
          qa[ks][2] = is0 ? *reinterpret_cast<const unsigned*>(q0 + ks * 16 + 8) : 0u;
          qa[ks][3] = is1 ? *reinterpret_cast<const unsigned*>(q1 + ks * 16 + 8) : 0u;
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        m_run[0] = m_run[1] = -INFINITY;
        l_run[0] = l_run[1] = 0.f;  // this lane's share of the row sums
      }
      if (!ring.wait(s)) return;
#pragma unroll 1
      for (int key0 = 0; key0 < SR; key0 += 16) {
        const int n_valid = u.keys - key0;  // keys from here on
        if (n_valid <= 0) break;
        if (!(u.pages >> (key0 / 16) & 1u)) continue;
        const unsigned kt = k_row + 2 * slot * C::kTileBytes + key0 * kBoxBytes, vt = v_row + 2 * slot * C::kTileBytes + key0 * kBoxBytes;
        if (n_valid < 16) {
          // what a page holds behind the sequence's end has weight 0, but may be anything: out of V's rows with it
          const unsigned v_tile = ring.tiles + (2 * slot + 1) * C::kTileBytes;
          for (int i = lane; i < (16 - n_valid) * C::kBoxes * kBoxPieces; i += 32)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             v_tile + (i / kBoxPieces % C::kBoxes * SR + key0 + n_valid + i / kBoxPieces / C::kBoxes) * kBoxBytes + i % kBoxPieces * 16),
                         "r"(0)
                         : "memory");
          __syncwarp();
        }
        // S = Q K^T for 16 keys: s0 = keys 0..7, s1 = keys 8..15
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          unsigned kb[4];
          ldmatrix_x4(kb, kt + ks / kSteps * (SR * kBoxBytes) + k_off[ks % kSteps]);
          mma16816<T>(s0, qa[ks], kb[0], kb[1]);
          mma16816<T>(s1, qa[ks], kb[2], kb[3]);
        }
        float v[8] = {s0[0], s0[1], s1[0], s1[1], s0[2], s0[3], s1[2], s1[3]};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int col = ((i >> 1) & 1) * 8 + 2 * tq + (i & 1);
          v[i] = col < n_valid ? v[i] * a.scale_log2 : -INFINITY;
        }
        float mx0 = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        float mx1 = fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7]));
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        if (__any_sync(0xffffffffu, mx0 > m_run[0] || mx1 > m_run[1])) {  // rare after the first stages
          const float mn0 = fmaxf(m_run[0], mx0), mn1 = fmaxf(m_run[1], mx1);
          const float a0 = m_run[0] == -INFINITY ? 0.f : ex2(m_run[0] - mn0);
          const float a1 = m_run[1] == -INFINITY ? 0.f : ex2(m_run[1] - mn1);
          l_run[0] = m_run[0] == -INFINITY ? l_run[0] : l_run[0] * a0;  // (0, or NaN to keep)
          l_run[1] = m_run[1] == -INFINITY ? l_run[1] : l_run[1] * a1;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][0] *= a0;
            o[n][1] *= a0;
            o[n][2] *= a1;
            o[n][3] *= a1;
          }
          m_run[0] = mn0;
          m_run[1] = mn1;
        }
        const float ms0 = m_run[0] == -INFINITY ? 0.f : m_run[0];
        const float ms1 = m_run[1] == -INFINITY ? 0.f : m_run[1];
        float p[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = ex2(v[i] - ms0);
          p[4 + i] = ex2(v[4 + i] - ms1);
        }
        l_run[0] += (p[0] + p[1]) + (p[2] + p[3]);
        l_run[1] += (p[4] + p[5]) + (p[6] + p[7]);
        // P as the A fragment of the second product, rounded to the cache's type as the products want it (l above is not): with the
        // rounding of the result that makes 1.2 to 1.4 times the distance from 64 bits that the latter alone makes. In fp16 a weight
        // of less than 2^-25 of the largest so far counts in l alone.
        unsigned pa[4];
        pa[0] = pack_pair<T>(p[0], p[1]);
        pa[1] = pack_pair<T>(p[4], p[5]);
        pa[2] = pack_pair<T>(p[2], p[3]);
        pa[3] = pack_pair<T>(p[6], p[7]);
#pragma unroll
        for (int c2 = 0; c2 < D / 16; ++c2) {
          unsigned vb[4];
          ldmatrix_x4_trans(vb, vt + c2 / kSteps * (SR * kBoxBytes) + v_off[c2 % kSteps]);
          mma16816<T>(o[2 * c2], pa, vb[0], vb[1]);
          mma16816<T>(o[2 * c2 + 1], pa, vb[2], vb[3]);
        }
        if (n_valid < 16) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next copy lands behind those zeros
      }
      __syncwarp();
      if (s > 0) ring.copy_next((s - 1) % C::kStages);
      if (u.last) {
        const size_t part = (static_cast<size_t>(blockIdx.x) * C::kWarps + warp + u.uid) * a.rs;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float l = l_run[i];
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          const int r = g + 8 * i;
          int b, h;
          if (!unit_row<RU>(a, u, r, &b, &h)) continue;
          if (u.last == 2) {
            const size_t row = static_cast<size_t>(b) * a.H + h;
            const float inv = l == 0.f ? 0.f : 1.f / l;  // (no key seen: O is 0 as well)
            T* const dst = static_cast<T*>(a.out) + row * D + 2 * tq;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
              *reinterpret_cast<unsigned*>(dst + n * 8) = pack_pair<T>(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
            if (a.lse && tq == 0) a.lse[row] = l > 0.f ? m_run[i] * kLn2 + logf(l) : l == 0.f ? -INFINITY : l;
          } else {
            float* const dst = a.part_o + (part + r) * D + 2 * tq;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            if (tq == 0) a.part_ml[part + r] = make_float2(m_run[i], l);
          }
        }
      }
    }
  });
}

// ---- fp32 caches --------------------------------------------------------------------

// kParts lanes share out a key's row and have their pieces of all query rows in registers. A step's partial sums, of RU rows for
// 32 / kParts keys, go through one butterfly that halves the rows of a lane at each exchange, so a lane ends with one row's score of
// one key, and keeps that row's maximum and sum. The weights go through shared memory to the lanes that have the columns of V.
template <int D, int kRows>
struct F32Cfg {
  // (eight rows: half the exchanges with eight lanes to a key, as far as the registers go: 64 heads on 8, 16384 rows of 128 87 -> 85 us)
  static constexpr int kWant = kRows == 1 ? 4 : kRows == 8 && D <= 128 ? 8 : 2 * kRows;
  static constexpr int kParts = kWant < D / 4 ? kWant : D / 4;
  static constexpr int kExtraBytes = (8 * 2 + 2) * kRows * 4;  // weights of 8 keys, each twice, and a factor a row, twice
  using Block = PagedBlock<float, D, kRows, (kExtraBytes + 15) & ~15>;
};

template <int D, int kRows>
__global__ void __launch_bounds__(F32Cfg<D, kRows>::Block::kThreads, 2) paged_f32_kernel(const __grid_constant__ PagedArgs a) {
  using C = typename F32Cfg<D, kRows>::Block;
  using tcgen::ffma2;
  constexpr int SR = C::SR, RU = C::RU, kVec = D / 4;
  constexpr int kKeys = 8, kParts = F32Cfg<D, kRows>::kParts;
  constexpr int kAtOnce = 32 / kParts, kSteps = kKeys / kAtOnce, kPieces = kVec / kParts;
  constexpr int kCols = kVec < 32 ? kVec : 32;           // lanes side by side on a row of V
  constexpr int kAt = 32 / kCols, kEach = kVec / kCols;  // rows of V at a time, 16-byte pieces of one a lane
  extern __shared__ __align__(1024) unsigned char smem[];
  paged_block<C>(a, nullptr, nullptr, smem, [&](Ring<C>& ring, int warp) {
    float2* const p_s = reinterpret_cast<float2*>(smem + C::kOffExtra + warp * ((F32Cfg<D, kRows>::kExtraBytes + 15) & ~15));  // [key][row]
    float2* const f_s = p_s + kKeys * RU;
    const unsigned char* const tiles = smem + warp * C::kRingBytes;
    const int lane = threadIdx.x & 31;
    const int part = lane % kParts, key_at = lane / kParts;  // scores
    const int col = lane % kCols, sub = lane / kCols;        // sum over V
    // the row whose scores the butterfly leaves here
    int my_row = 0;
#pragma unroll
    for (int d = 1, n = RU; d < kParts; d *= 2)
      if (n > 1) {
        n /= 2;
        if (lane & d) my_row += n;
      }
    // Pieces of a lane: every kParts-th. With four lanes to a key, eight neighbouring lanes have two keys, whose rows begin in the same
    // bank, so those of odd keys take the other half of each group of eight pieces first.
    auto piece = [&](int j) { return (j * kParts + part) ^ (kParts == 4 ? (key_at & 1) * 4 : 0); };
    float4 q[RU][kPieces];
    float2 o[RU][kEach][2];
    float m_run = -INFINITY, l_run = 0.f;
    const int total = ring.total;
    for (int s = 0; s < total; ++s) {
      const int slot = s % C::kStages;
      const StageInfo u = ring.info[slot];
      if (u.first) {  // (while the copy is on its way)
#pragma unroll
        for (int r = 0; r < RU; ++r) {
          int b, h;
          const bool is = unit_row<RU>(a, u, r, &b, &h);
          const float4* const src = static_cast<const float4*>(a.q) + (is ? static_cast<size_t>(b) * a.H + h : 0) * kVec;
#pragma unroll
          for (int j = 0; j < kPieces; ++j) q[r][j] = is ? src[piece(j)] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int e = 0; e < kEach; ++e) o[r][e][0] = o[r][e][1] = make_float2(0.f, 0.f);
        }
        m_run = -INFINITY;
        l_run = 0.f;
      }
      if (!ring.wait(s)) return;
#pragma unroll 1
      for (int key0 = 0; key0 < SR; key0 += kKeys) {
        const int n_valid = u.keys - key0;
        if (n_valid <= 0) break;
        if (!(u.pages >> (key0 / 16) & 1u)) continue;
        const unsigned char* const kt = tiles + 2 * slot * C::kTileBytes + key0 * C::kRowBytes;
        const unsigned char* const vt = tiles + (2 * slot + 1) * C::kTileBytes + key0 * C::kRowBytes;
        float sc[kSteps];
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const float4* const row = reinterpret_cast<const float4*>(kt + (st * kAtOnce + key_at) * C::kRowBytes);
          float2 acc[RU];
#pragma unroll
          for (int r = 0; r < RU; ++r) acc[r] = make_float2(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < kPieces; ++j) {
            const float4 x = row[piece(j)];
#pragma unroll
            for (int r = 0; r < RU; ++r) {
              acc[r] = ffma2(make_float2(x.x, x.y), make_float2(q[r][j].x, q[r][j].y), acc[r]);
              acc[r] = ffma2(make_float2(x.z, x.w), make_float2(q[r][j].z, q[r][j].w), acc[r]);
            }
          }
          float v[RU];
#pragma unroll
          for (int r = 0; r < RU; ++r) v[r] = acc[r].x + acc[r].y;
#pragma unroll
          for (int d = 1, n = RU; d < kParts; d *= 2) {
            if (n > 1) {
              n /= 2;
              const bool upper = (lane & d) != 0;
#pragma unroll
              for (int r = 0; r < RU / 2; ++r) {
                if (r >= n) break;
                const float keep = upper ? v[r + n] : v[r], give = upper ? v[r] : v[r + n];
                v[r] = keep + __shfl_xor_sync(0xffffffffu, give, d);
              }
            } else {
              v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
            }
          }
          sc[st] = st * kAtOnce + key_at < n_valid ? v[0] * a.scale_log2 : -INFINITY;
        }
        // this lane's row: maximum over the stage's keys
        float mx = sc[0];
#pragma unroll
        for (int st = 1; st < kSteps; ++st) mx = fmaxf(mx, sc[st]);
#pragma unroll
        for (int d = kParts; d < 32; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        if (__any_sync(0xffffffffu, mx > m_run)) {
          const float mn = fmaxf(m_run, mx);
          const float f = m_run == -INFINITY ? 0.f : ex2(m_run - mn);
          l_run = m_run == -INFINITY ? l_run : l_run * f;  // (0, or NaN to keep)
          m_run = mn;
          __syncwarp();
          if (key_at == 0) f_s[my_row] = make_float2(f, f);
          __syncwarp();
#pragma unroll
          for (int r = 0; r < RU; ++r) {
            const float2 g = f_s[r];
#pragma unroll
            for (int e = 0; e < kEach; ++e)
#pragma unroll
              for (int i = 0; i < 2; ++i) o[r][e][i] = make_float2(o[r][e][i].x * g.x, o[r][e][i].y * g.x);
          }
        }
        const float ms = m_run == -INFINITY ? 0.f : m_run;
        __syncwarp();  // the weights of the keys before have been read
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const float p = ex2(sc[st] - ms);
          l_run += p;
          p_s[(st * kAtOnce + key_at) * RU + my_row] = make_float2(p, p);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kKeys / kAt; ++i) {
          const int row = i * kAt + sub;
          if (row < n_valid) {  // (rows behind the end may hold anything)
            float4 x[kEach];
#pragma unroll
            for (int e = 0; e < kEach; ++e) x[e] = reinterpret_cast<const float4*>(vt + row * C::kRowBytes)[e * kCols + col];
#pragma unroll
            for (int r = 0; r < RU; ++r) {
              const float2 p = p_s[row * RU + r];
#pragma unroll
              for (int e = 0; e < kEach; ++e) {
                o[r][e][0] = ffma2(p, make_float2(x[e].x, x[e].y), o[r][e][0]);
                o[r][e][1] = ffma2(p, make_float2(x[e].z, x[e].w), o[r][e][1]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (s > 0) ring.copy_next((s - 1) % C::kStages);
      if (u.last) {
        const size_t at = (static_cast<size_t>(blockIdx.x) * C::kWarps + warp + u.uid) * a.rs;
        float l_of = l_run;
#pragma unroll
        for (int d = kParts; d < 32; d *= 2) l_of += __shfl_xor_sync(0xffffffffu, l_of, d);
        __syncwarp();
        if (key_at == 0) f_s[my_row] = make_float2(m_run, l_of);
        __syncwarp();
#pragma unroll
        for (int r = 0; r < RU; ++r) {
#pragma unroll
          for (int e = 0; e < kEach; ++e)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int d = kCols; d < 32; d *= 2) {
                o[r][e][i].x += __shfl_xor_sync(0xffffffffu, o[r][e][i].x, d);
                o[r][e][i].y += __shfl_xor_sync(0xffffffffu, o[r][e][i].y, d);
              }
          int b, h;
          if (!unit_row<RU>(a, u, r, &b, &h) || sub != 0) continue;
          const float2 ml = f_s[r];
          const bool result = u.last == 2;
          const size_t row = static_cast<size_t>(b) * a.H + h;
          const float f = !result ? 1.f : ml.y == 0.f ? 0.f : 1.f / ml.y;  // (no key seen: O is 0 as well)
          float4* const dst = reinterpret_cast<float4*>(result ? static_cast<float*>(a.out) + row * D : a.part_o + (at + r) * D);
#pragma unroll
          for (int e = 0; e < kEach; ++e)
            dst[e * kCols + col] = make_float4(o[r][e][0].x * f, o[r][e][0].y * f, o[r][e][1].x * f, o[r][e][1].y * f);
          if (lane == 0 && !result) a.part_ml[at + r] = ml;
          if (lane == 0 && result && a.lse) a.lse[row] = ml.y > 0.f ? ml.x * kLn2 + logf(ml.y) : ml.y == 0.f ? -INFINITY : ml.y;
        }
      }
    }
  });
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

// ---- host side ----------------------------------------------------------------------

constexpr int kBlocksPerSm = 2;  // of both kernels

int fp32_rows(int G) { return G <= 1 ? 1 : G <= 2 ? 2 : G <= 4 ? 4 : 8; }

// How a call runs, and its room: which shares have parts of a unit, and (m, l) and O of every part. A share leaves at most one
// part of a unit, and share c's of unit u is part c + u: both only grow along the list, so no two meet.
struct PagedPlan {
  int RU, SR, HB, RB, warps, blocks;  // (warps of a block)
  int rs;       // rows of a part
  double most;  // stages that there can be
  bool listed;  // shared pages by every sequence for itself, the batch being small
  bool tc;      // shared pages by the tensor-core kernel (32 sequences on 32768 rows, H32/kvH8 D128: 323 us without, 57 with it)
  SharedPlan shared;
  size_t unit_bytes, ml_bytes, o_bytes, shared_ml_bytes, bytes;
};

// 16 bits: where the batch would read no more than this over again, every sequence reads the shared pages for itself, out of the L2
// but for the first, and the call has one kernel less in its chain. us on the device, by every sequence / once: H32/kvH8 D128, 2 sequences
// on 2048 shared rows (8 MB over again) 12.5 / 15.9, on 4096 (17 MB) 14.9 / 17.7, 64 on 64 (17 MB) 12.3 / 16.0, 32 on 256 (33 MB) 13.8 /
// 13.2; 200 on 512, H16/kvH4 D32 (52 MB) 21.7 / 17.5.
constexpr double kListedBytes = 28e6;

PagedPlan make_plan(const ra_paged_kv& c, int heads, int shared_len) {
  PagedPlan p = {};
  const int G = (heads + c.kv_heads - 1) / c.kv_heads;
  const bool f32 = c.dtype == RA_F32;
  p.listed = !f32 && shared_len > 0 && 4.0 * (c.batch - 1) * shared_len * c.kv_heads * c.head_dim <= kListedBytes;
  if (p.listed) shared_len = 0;
  const long long rows_shared = shared_len > 0 ? static_cast<long long>(c.batch) * G : 0;
  p.RU = f32 ? fp32_rows(static_cast<int>(std::max<long long>(std::min<long long>(rows_shared, 8), G))) : kMmaRows;
  p.SR = stage_keys(f32, c.head_dim);
  p.warps = block_warps(f32, c.head_dim);
  p.tc = !f32 && rows_shared > 0 && plan_shared_prefix(c.batch, heads, c.kv_heads, c.head_dim, shared_len, &p.shared);
  p.HB = (G + p.RU - 1) / p.RU;
  p.RB = p.tc ? 0 : static_cast<int>((rows_shared + p.RU - 1) / p.RU);
  const size_t units = static_cast<size_t>(c.kv_heads) * (p.RB + static_cast<size_t>(c.batch) * p.HB);
  // as many stages as the tables have room for
  const long long room = static_cast<long long>(c.max_pages) * c.page_size;
  p.most = static_cast<double>(c.kv_heads) * (static_cast<double>(c.batch) * p.HB * ((room + p.SR - 1) / p.SR) +
                                              static_cast<double>(p.RB) * ((shared_len + p.SR - 1) / p.SR));
  const int wave = kBlocksPerSm * sm_count();
  p.blocks = p.most < static_cast<double>(wave) * p.warps ? (static_cast<int>(p.most) + p.warps - 1) / p.warps : wave;
  p.rs = p.RB > 0 ? p.RU : std::min(p.RU, G);
  auto whole = [](size_t n) { return (n + 127) & ~static_cast<size_t>(127); };
  const size_t rows = (units + static_cast<size_t>(p.blocks) * p.warps) * p.rs, shared_rows = p.tc ? shared_part_rows(p.shared, c.kv_heads) : 0;
  p.unit_bytes = whole(units * sizeof(int2));
  p.ml_bytes = whole(rows * sizeof(float2));
  p.o_bytes = whole(rows * c.head_dim * sizeof(float));
  p.shared_ml_bytes = whole(shared_rows * sizeof(float2));
  p.bytes = p.unit_bytes + p.ml_bytes + p.o_bytes + p.shared_ml_bytes + shared_rows * c.head_dim * sizeof(float);
  return p;
}

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

template <typename T, int D, int RU>
int launch_rows(const ra_paged_kv& c, const PagedArgs& a, const PagedPlan& p, cudaStream_t stream) {
  int rc = RA_OK;
  if constexpr (sizeof(T) == 4) {
    if (p.blocks > 0) rc = launch_main<paged_f32_kernel<D, RU>, typename F32Cfg<D, RU>::Block>(p.blocks, stream, a);
  } else if (p.blocks > 0) {
    CUtensorMap k, v;
    const long long heads = static_cast<long long>(a.num_pages) * a.kvH, stride = static_cast<long long>(c.page_size) * D;
    const int box = std::min(c.page_size, p.SR);
    rc = tcgen::make_map(&k, c.dtype, c.k, D, c.page_size, heads, stride, box, MmaBlock<T, D>::kBoxBytes);
    if (rc == RA_OK) rc = tcgen::make_map(&v, c.dtype, c.v, D, c.page_size, heads, stride, box, MmaBlock<T, D>::kBoxBytes);
    if (rc == RA_OK) rc = launch_main<paged_mma_kernel<T, D>, MmaBlock<T, D>>(p.blocks, stream, k, v, a);
  }
  if (rc != RA_OK) return rc;
  return launch_fold<T, D, RU>(a, stream);
}

template <int D>
int launch_head_dim(const ra_paged_kv& c, const PagedArgs& a, const PagedPlan& p, cudaStream_t stream) {
  if (c.dtype == RA_F16) return launch_rows<__half, D, kMmaRows>(c, a, p, stream);
  if (c.dtype == RA_BF16) return launch_rows<__nv_bfloat16, D, kMmaRows>(c, a, p, stream);
  if (p.RU == 1) return launch_rows<float, D, 1>(c, a, p, stream);
  if (p.RU == 2) return launch_rows<float, D, 2>(c, a, p, stream);
  if (p.RU == 4) return launch_rows<float, D, 4>(c, a, p, stream);
  return launch_rows<float, D, 8>(c, a, p, stream);
}

int check_decode(const ra_paged_kv& c, int heads, const int* shared_pages, int shared_len) {
  const char* const what = "paged_decode";
  RAB_REQUIRE(c.dtype == RA_F32 || c.dtype == RA_F16 || c.dtype == RA_BF16, RA_ERR_INVALID, "%s: unknown dtype %d", what, c.dtype);
  RAB_REQUIRE(c.head_dim == 32 || c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, RA_ERR_UNSUPPORTED,
              "%s: unsupported head_dim=%d (supported: 32, 64, 128, 256)", what, c.head_dim);
  const int rc = check_paged(c, what);
  if (rc != RA_OK) return rc;
  RAB_REQUIRE(heads >= c.kv_heads && heads <= 4096, RA_ERR_INVALID, "%s: bad heads", what);
  RAB_REQUIRE(static_cast<long long>(c.batch) * heads < (1ll << 24), RA_ERR_INVALID, "%s: too many rows", what);
  RAB_REQUIRE(static_cast<long long>(c.num_pages) * c.kv_heads < (1ll << 31) - 1, RA_ERR_INVALID, "%s: too many pages", what);
  RAB_REQUIRE(shared_len >= 0 && shared_len % c.page_size == 0 && (shared_len == 0 || shared_pages), RA_ERR_INVALID,
              "%s: shared pages are whole: shared_len=%d, page_size=%d", what, shared_len, c.page_size);
  RAB_REQUIRE(shared_len <= 1 << 30, RA_ERR_INVALID, "%s: shared_len=%d is above 2^30", what, shared_len);
  return RA_OK;
}

// A cache without pages holds no keys, whatever the tables say.
ra_paged_kv without_pages(ra_paged_kv c, int* shared_len) {
  if (c.num_pages == 0) c.max_pages = *shared_len = 0;
  return c;
}

}  // namespace
}  // namespace rab

using namespace rab;

extern "C" {

size_t ra_paged_decode_workspace_bytes(const ra_paged_kv* cache, int heads, int shared_len) {
  int none = 0;
  if (!cache || check_decode(*cache, heads, &none, shared_len) != RA_OK) return 0;
  const ra_paged_kv c = without_pages(*cache, &shared_len);
  return make_plan(c, heads, shared_len).bytes;
}

int ra_debug_paged_route(const ra_paged_kv* cache, int heads, int shared_len) {
  int none = 0;
  if (!cache || check_decode(*cache, heads, &none, shared_len) != RA_OK) return -1;
  const ra_paged_kv c = without_pages(*cache, &shared_len);
  const PagedPlan p = make_plan(c, heads, shared_len);
  return shared_len == 0 ? 0 : p.listed ? 1 : p.tc ? 3 : 2;
}

int ra_paged_decode(const ra_paged_kv* cache, const void* q, int heads, const int* shared_pages, int shared_len, void* out,
                    float* lse, void* workspace, size_t workspace_bytes, ra_stream stream_) {
  RAB_REQUIRE(cache != nullptr, RA_ERR_INVALID, "paged_decode: null argument");
  int rc = check_decode(*cache, heads, shared_pages, shared_len);
  if (rc == RA_OK) rc = check_lists(*cache, "paged_decode");
  if (rc != RA_OK) return rc;
  if (cache->batch == 0) return RA_OK;
  RAB_REQUIRE(q && out, RA_ERR_INVALID, "paged_decode: null argument");
  RAB_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0, RA_ERR_INVALID,
              "paged_decode: q and out must be 16-byte aligned");
  RAB_REQUIRE(((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(shared_pages)) & 3u) == 0, RA_ERR_INVALID,
              "paged_decode: lse or shared_pages is not aligned to its elements");
  const ra_paged_kv c = without_pages(*cache, &shared_len);
  const PagedPlan p = make_plan(c, heads, shared_len);
  // (a share is counted in 32 bits; tables that name a page over and over could ask for more)
  RAB_REQUIRE(p.most < 2147483648.0 * std::max(p.blocks * p.warps, 1), RA_ERR_INVALID, "paged_decode: too many keys");
  RAB_REQUIRE(workspace && workspace_bytes >= p.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, RA_ERR_OVERFLOW,
              "paged_decode: workspace too small or not 16-byte aligned");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  unsigned char* const ws = static_cast<unsigned char*>(workspace);
  PagedArgs a;
  a.q = q;
  a.k = c.k;
  a.v = c.v;
  a.out = out;
  a.lse = lse;
  a.table = c.page_table;
  a.table_stride = c.table_stride;
  a.lens = c.lens;
  a.shared_pages = shared_pages;
  a.shared_len = p.listed ? 0 : shared_len;
  a.listed_len = p.listed ? shared_len : 0;
  a.num_pages = c.num_pages;
  a.max_pages = c.max_pages;
  a.shift = page_shift(c.page_size);
  a.B = c.batch;
  a.H = heads;
  a.kvH = c.kv_heads;
  a.G = (heads + c.kv_heads - 1) / c.kv_heads;
  a.HB = p.HB;
  a.RB = p.RB;
  a.rs = p.rs;
  a.scale_log2 = kLog2e / std::sqrt(static_cast<float>(c.head_dim));
  a.unit_parts = reinterpret_cast<int2*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + p.unit_bytes);
  a.part_o = reinterpret_cast<float*>(ws + p.unit_bytes + p.ml_bytes);
  a.shared = p.shared;
  a.shared_ml = nullptr;
  a.shared_o = nullptr;
  a.status = device_status_ptr();
  RAB_REQUIRE(a.status != nullptr, RA_ERR_CUDA, "paged_decode: no device status word");
  a.wait_ns = tcgen::tc_wait_limit_ns();
  a.shares = p.blocks * p.warps;
  const int stall = tcgen::tc_stall_after();
  a.missing = stall > 0 ? 16 : stall == 0 ? -1 : 0;
  if (p.tc) {
    a.shared_ml = reinterpret_cast<float2*>(ws + p.unit_bytes + p.ml_bytes + p.o_bytes);
    a.shared_o = reinterpret_cast<float*>(ws + p.unit_bytes + p.ml_bytes + p.o_bytes + p.shared_ml_bytes);
    const SharedPrefix s{q, c.k, c.v, a.B, a.H, a.kvH, c.head_dim, shared_pages, c.lens, shared_len, c.num_pages, c.max_pages, a.shift};
    rc = launch_shared_prefix(c.dtype, s, p.shared, a.shared_o, a.shared_ml, stream);
    if (rc != RA_OK) return rc;
  }
  if (c.head_dim == 32) return launch_head_dim<32>(c, a, p, stream);
  if (c.head_dim == 64) return launch_head_dim<64>(c, a, p, stream);
  if (c.head_dim == 128) return launch_head_dim<128>(c, a, p, stream);
  return launch_head_dim<256>(c, a, p, stream);
}

}  // extern "C"
