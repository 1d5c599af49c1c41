// Decode attention (one query row a sequence) against a paged KV cache, sequences of any lengths, which only the device knows;
// and for a batch whose sequences begin with the same pages, those once for all.
//
//   out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(q . k_j / sqrt(D)),  j < lens[b],  KV head h % kv_heads
//
// What bounds it is the cache: every row is read once. The work is cut into units, the up to RU query rows that read the same
// keys: the heads of a KV head and a sequence, behind the shared pages where the sequence has them; and for the shared pages RU
// rows of all sequences. A unit is a list of stages of SR keys, and all units' stages one after the other are dealt in equal
// shares to the blocks of one wave, so that lengths do not matter to the balance. A block streams its share through a
// shared-memory ring without a pause where units meet (16-byte cp.async; page numbers are read a stage ahead). A unit that lies in one
// share is finished there; of others every share leaves (O, m, l) in the workspace, and a second kernel folds them.
//
// 16-bit caches: both products on mma.sync m16n8k16, the unit's rows as its M rows, as in decode_mma_kernel (decode.cu). fp32:
// plain multiply-adds, the scores of a stage by groups of lanes and its values by columns.
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
  int shared_len;  // rows in shared pages
  int num_pages, max_pages, shift;
  int B, H, kvH;
  int G;          // heads of a KV head, at most
  int HB;         // units of a KV head and a sequence
  int RB;         // units of a KV head on the shared pages (0: not by this kernel)
  int rs;         // rows of a part in the workspace
  int min_per;    // stages of a share, at least
  float scale_log2;
  long long* head;  // {stages of a share, first stage of every sequence}
  float2* part_ml;  // (m in log2 units, l) of rs rows, a part after the other
  float* part_o;
  // shared pages by the tensor-core kernel (step_tc.cu; RB is 0 then): its parts, see SharedPrefix
  SharedPlan shared;
  float2* shared_ml;  // NULL: not by it
  float* shared_o;
  const int* status;
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
  int uid;          // number of the unit; units on the shared pages come first
  int b, kvh, hb;   // b = -1: on the shared pages
  int st, n;        // stage of the unit and how many it has
  int start, end;   // its keys
  __device__ inline int prefix_stages(const PagedArgs& a) const { return (a.shared_len + SR - 1) / SR; }
  __device__ inline void on_shared(const PagedArgs& a) {
    b = -1;
    start = 0;
    end = a.shared_len;
    n = prefix_stages(a);
  }
  __device__ inline void on_sequence(const PagedArgs& a, int seq) {
    b = seq;
    own_keys(a, b, &start, &end);
    n = static_cast<int>((static_cast<long long>(end) - start + SR - 1) / SR);
  }
  __device__ inline void number(const PagedArgs& a) { uid = b < 0 ? kvh * a.RB + hb : a.kvH * a.RB + (b * a.kvH + kvh) * a.HB + hb; }
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

// Sum over the block of a thread's v, and the sum over the threads before it.
template <int kThreads>
__device__ inline long long block_scan(long long v, long long* total, long long* room) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = v;
#pragma unroll
  for (int i = 1; i < 32; i *= 2) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, i);
    if (lane >= i) incl += o;
  }
  __syncthreads();
  if (lane == 31) room[warp] = incl;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += room[w];
    all += room[w];
  }
  *total = all;
  return before + incl - v;
}

// The block's share: its first place and how many stages; *per: stages of a share. Block 0 writes the head of the workspace.
template <int SR, int kThreads>
__device__ inline int find_share(const PagedArgs& a, Walk<SR>* w, long long* per) {
  __shared__ long long room[kThreads / 32];
  __shared__ int seq;
  __shared__ long long in_seq;
  const int units = a.kvH * a.HB;
  long long shared_total = 0;
  if (a.RB > 0) shared_total = static_cast<long long>(a.kvH) * a.RB * w->prefix_stages(a);
  // the first chunk of sequences stays at hand
  const int mine = static_cast<int>(threadIdx.x) < a.B ? own_stages<SR>(a, threadIdx.x) : 0;
  long long sum = mine, total;
  for (int b = static_cast<int>(threadIdx.x) + kThreads; b < a.B; b += kThreads) sum += own_stages<SR>(a, b);
  block_scan<kThreads>(sum, &total, room);
  const long long all = shared_total + total * units;
  *per = max(static_cast<long long>(a.min_per), (all + gridDim.x - 1) / gridDim.x);
  const long long first = *per * blockIdx.x, stages = min(*per, all - first);
  const bool writer = blockIdx.x == 0;
  if (writer && threadIdx.x == 0) a.head[0] = *per;
  if (stages <= 0 && !writer) return 0;
  const bool on_shared = first < shared_total;
  if (!on_shared || writer) {
    long long base = shared_total;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
      const int b = b0 + static_cast<int>(threadIdx.x);
      const long long n = (b0 == 0 ? mine : b < a.B ? own_stages<SR>(a, b) : 0) * static_cast<long long>(units);
      long long chunk;
      const long long at = base + block_scan<kThreads>(n, &chunk, room);
      if (writer && b < a.B) a.head[1 + b] = at;
      if (first >= at && first < at + n) {
        seq = b;
        in_seq = first - at;
      }
      base += chunk;
      if (!writer && first < base) break;
    }
    __syncthreads();
  }
  if (stages <= 0) return 0;
  if (on_shared) {
    w->on_shared(a);
    const int u = static_cast<int>(first / w->n);
    w->st = static_cast<int>(first - static_cast<long long>(u) * w->n);
    w->kvh = u / a.RB;
    w->hb = u % a.RB;
  } else {
    w->on_sequence(a, seq);
    const int u = static_cast<int>(in_seq / w->n);
    w->st = static_cast<int>(in_seq - static_cast<long long>(u) * w->n);
    w->kvh = u / a.HB;
    w->hb = u % a.HB;
  }
  w->number(a);
  return static_cast<int>(stages);
}

// Behind the kernel of the shared pages, whose blocks let this one begin when all that came before them has completed, nothing
// waits for that kernel itself but the end: the fold, which waits for this grid, then finds both kernels' parts.
__device__ inline void begin_main(const PagedArgs& a) {
  let_next_start();
  if (a.shared_ml == nullptr) wait_for_previous();
}
__device__ inline void end_main(const PagedArgs& a) {
  if (a.shared_ml != nullptr) wait_for_previous();
}

// Query row r of a unit: sequence and head; false where the unit has no such row.
template <int RU, int SR>
__device__ inline bool unit_row(const PagedArgs& a, const Walk<SR>& w, int r, int* b, int* h) {
  const int i = w.hb * RU + r, g = w.b < 0 ? i % a.G : i;
  *b = w.b < 0 ? i / a.G : w.b;
  *h = w.kvh + a.kvH * g;
  return *b < a.B && *h < a.H;
}

// Row indexes in the cache of the 16-key blocks of a stage (-1: none), and the asynchronous copies of a stage.
template <typename T, int D, int SR, int kThreads>
struct Loader {
  static constexpr int kPieces = D * static_cast<int>(sizeof(T)) / 16;
  static constexpr int kBlocks = SR / 16;
  long long at[kBlocks];
  // a 16-byte piece's place in its row, so that neither the rows of an ldmatrix nor the lanes that share out a row meet in a bank
  __device__ static inline int place(int r, int c) {
    if constexpr (sizeof(T) == 4) return c ^ ((r & 1) << 2);
    else return kPieces == 4 ? c ^ ((r >> 1) & 3) : c ^ (r & 7);
  }
  __device__ inline void look_up(const PagedArgs& a, const Walk<SR>& w) {
    const int* table = w.b < 0 ? a.shared_pages : a.table + w.b * a.table_stride;
    const int most = w.b < 0 ? a.shared_len >> a.shift : a.max_pages;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const long long slot = static_cast<long long>(w.start) + static_cast<long long>(w.st) * SR + 16 * i;
      const long long row = slot < w.end ? paged_row(table, most, a.num_pages, a.shift, a.kvH, slot) : -1;
      at[i] = row < 0 ? -1 : row + (static_cast<long long>(w.kvh) << a.shift);
    }
  }
  __device__ inline void issue(const PagedArgs& a, const Walk<SR>& w, unsigned char* k_slot, unsigned char* v_slot, int* ok) const {
    const int tid = threadIdx.x;
    const int left = w.end - w.start - w.st * SR;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
      if (tid == i) ok[i] = at[i] >= 0;
#pragma unroll
    for (int i = 0; i < SR * kPieces / kThreads; ++i) {
      const int p = tid + i * kThreads, r = p / kPieces, c = p % kPieces;
      long long row = at[0];
#pragma unroll
      for (int j = 1; j < kBlocks; ++j) row = (r >> 4) == j ? at[j] : row;
      const bool there = row >= 0 && r < left;
      const size_t off = there ? (static_cast<size_t>(row + (r & 15)) * kPieces + c) * 16 : 0;
      const int dst = (r * kPieces + place(r, c)) * 16;
      cp_async16(k_slot + dst, static_cast<const unsigned char*>(a.k) + off, there ? 16 : 0);
      cp_async16(v_slot + dst, static_cast<const unsigned char*>(a.v) + off, there ? 16 : 0);
    }
  }
};

template <typename T>
__device__ inline void put4(T* dst, float4 v);
template <>
__device__ inline void put4<float>(float* dst, float4 v) {
  *reinterpret_cast<float4*>(dst) = v;
}
template <>
__device__ inline void put4<__half>(__half* dst, float4 v) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_pair<__half>(v.x, v.y), pack_pair<__half>(v.z, v.w));
}
template <>
__device__ inline void put4<__nv_bfloat16>(__nv_bfloat16* dst, float4 v) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_pair<__nv_bfloat16>(v.x, v.y), pack_pair<__nv_bfloat16>(v.z, v.w));
}

// The end of a unit, or of the block's part of it: `rows` rows of (m, l) and O in shared memory, O relative to m and summed over
// nothing any more. A unit that the block has whole, and no shared pages ahead of it, is the result; others go to the workspace.
template <typename T, int D, int RU, int SR, int kThreads>
__device__ inline void put_unit(const PagedArgs& a, const Walk<SR>& w, bool whole, const float* m, const float* l, const float* o) {
  constexpr int kVec = D / 4;
  const bool direct = whole && w.b >= 0 && w.start == 0;
  const size_t part = (static_cast<size_t>(blockIdx.x) + w.uid) * a.rs;
  for (int i = threadIdx.x; i < RU * kVec; i += kThreads) {
    const int r = i / kVec, col = i % kVec * 4;
    int b, h;
    if (!unit_row<RU>(a, w, r, &b, &h)) continue;
    float4 v = *reinterpret_cast<const float4*>(o + r * D + col);
    if (direct) {
      const float inv = l[r] > 0.f ? 1.f / l[r] : 0.f;
      const size_t row = static_cast<size_t>(b) * a.H + h;
      put4(static_cast<T*>(a.out) + row * D + col, l[r] == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                                              : make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
      if (a.lse && col == 0) a.lse[row] = l[r] > 0.f ? m[r] * kLn2 + logf(l[r]) : l[r] == 0.f ? -INFINITY : l[r];
    } else {
      *reinterpret_cast<float4*>(a.part_o + (part + r) * D + col) = v;
      if (col == 0) a.part_ml[part + r] = make_float2(m[r], l[r]);
    }
  }
}

// ---- 16-bit caches ------------------------------------------------------------------

template <int D>
struct PagedMma {
  static constexpr int RU = 16;
  static constexpr int kWarps = D == 256 ? 2 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int SR = kWarps * 16;
  static constexpr int kStageBytes = SR * D * 2;  // per tensor
  // 96 KB of ring and two blocks an SM, as in decode_mma_kernel
  static constexpr int kStages = 96 * 1024 / (2 * kStageBytes) < 8 ? 96 * 1024 / (2 * kStageBytes) : 8;
  static constexpr int kOffMerge = 2 * kStages * kStageBytes;
  static constexpr int kMergeRows = 16 * (kWarps / 2);
  static constexpr int kOffMl = kOffMerge + kMergeRows * D * 4;
  static constexpr int kOffOk = kOffMl + (kWarps + 1) * 32 * 4;
  static constexpr int kSmemBytes = kOffOk + kStages * (SR / 16) * 4;
};

template <typename T, int D>
__global__ void __launch_bounds__(PagedMma<D>::kThreads) paged_mma_kernel(PagedArgs a) {
  using C = PagedMma<D>;
  constexpr int SR = C::SR, RU = C::RU, kStages = C::kStages;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const k_ring = smem;
  unsigned char* const v_ring = smem + kStages * C::kStageBytes;
  float* const merge = reinterpret_cast<float*>(smem + C::kOffMerge);
  float* const red_m = reinterpret_cast<float*>(smem + C::kOffMl);  // [warps + 1][16], then l likewise
  float* const red_l = red_m + (C::kWarps + 1) * 16;
  int* const ok_ring = reinterpret_cast<int*>(smem + C::kOffOk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, tq = lane & 3;  // fragment row (and row + 8), column pair

  begin_main(a);
  Walk<SR> wc;
  long long per;
  const int total = find_share<SR, C::kThreads>(a, &wc, &per);
  if (total == 0) {
    end_main(a);
    return;
  }
  Walk<SR> wi = wc;  // ahead of wc by what the ring holds
  Loader<T, D, SR, C::kThreads> load;
  load.look_up(a, wi);
  int issued = 0;
  auto issue = [&]() {
    if (issued < total) {
      const int slot = issued % kStages;
      load.issue(a, wi, k_ring + slot * C::kStageBytes, v_ring + slot * C::kStageBytes, ok_ring + slot * (SR / 16));
      if (++issued < total) {
        wi.next(a);
        load.look_up(a, wi);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue();

  unsigned qa[D / 16][4];
  float o[D / 8][4];
  float m_run[2], l_run[2];
  const int mi = lane >> 3, r8 = lane & 7, key0 = warp * 16;
  const unsigned k_row_off = static_cast<unsigned>((key0 + (mi >> 1) * 8 + r8) * D * 2);
  const unsigned v_row_off = static_cast<unsigned>((key0 + (mi & 1) * 8 + r8) * D * 2);
  int first_st = wc.st;  // first stage of the block's part of the unit
  for (int s = 0; s < total; ++s) {
    if (s == 0 || wc.st == 0) {
      first_st = wc.st;
      // Q as A fragments: reg0 (row g, k 2tq..), reg1 (row g+8, same k), reg2 / reg3 the same at k+8
      int b0, h0, b1, h1;
      const bool is0 = unit_row<RU>(a, wc, g, &b0, &h0), is1 = unit_row<RU>(a, wc, g + 8, &b1, &h1);
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
    cp_async_wait<kStages - 2>();
    __syncthreads();
    issue();
    const int slot = s % kStages;
    const int n_valid = wc.end - wc.start - wc.st * SR - key0;  // keys of this warp's block
    if (n_valid > 0 && ok_ring[slot * (SR / 16) + warp]) {
      const unsigned kt = static_cast<unsigned>(__cvta_generic_to_shared(k_ring + slot * C::kStageBytes));
      const unsigned vt = static_cast<unsigned>(__cvta_generic_to_shared(v_ring + slot * C::kStageBytes));
      // S = Q K^T for 16 keys: s0 = keys 0..7, s1 = keys 8..15
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        unsigned kb[4];
        ldmatrix_x4(kb, kt + k_row_off + (load.place(r8, 2 * ks + (mi & 1)) << 4));
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
      if (__any_sync(0xffffffffu, mx0 > m_run[0] || mx1 > m_run[1])) {  // rare after the first blocks
        const float mn0 = fmaxf(m_run[0], mx0), mn1 = fmaxf(m_run[1], mx1);
        const float a0 = m_run[0] == -INFINITY ? 0.f : ex2(m_run[0] - mn0);
        const float a1 = m_run[1] == -INFINITY ? 0.f : ex2(m_run[1] - mn1);
        l_run[0] *= a0;
        l_run[1] *= a1;
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
      // P as the A fragment of the second product, rounded to the cache's type as the products want it
      unsigned pa[4];
      pa[0] = pack_pair<T>(p[0], p[1]);
      pa[1] = pack_pair<T>(p[4], p[5]);
      pa[2] = pack_pair<T>(p[2], p[3]);
      pa[3] = pack_pair<T>(p[6], p[7]);
#pragma unroll
      for (int c2 = 0; c2 < D / 16; ++c2) {
        unsigned vb[4];
        ldmatrix_x4_trans(vb, vt + v_row_off + (load.place(r8, 2 * c2 + (mi >> 1)) << 4));
        mma16816<T>(o[2 * c2], pa, vb[0], vb[1]);
        mma16816<T>(o[2 * c2 + 1], pa, vb[2], vb[3]);
      }
    }
    if (wc.st == wc.n - 1 || s == total - 1) {
      // the lanes of a row, then the warps, in pairs: the upper half of the warps stages its O
      const bool whole = first_st == 0 && wc.st == wc.n - 1;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
        l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
      }
      if (tq == 0) {
        red_m[warp * 16 + g] = m_run[0];
        red_m[warp * 16 + g + 8] = m_run[1];
        red_l[warp * 16 + g] = l_run[0];
        red_l[warp * 16 + g + 8] = l_run[1];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float m_all = -INFINITY, l_all = 0.f;
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) m_all = fmaxf(m_all, red_m[w * 16 + g + 8 * i]);
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) {
          const float mw = red_m[w * 16 + g + 8 * i];
          l_all += (mw == -INFINITY ? (red_l[w * 16 + g + 8 * i] == 0.f ? 0.f : 1.f) : ex2(mw - m_all)) * red_l[w * 16 + g + 8 * i];
        }
        const float f = m_run[i] == -INFINITY ? 1.f : ex2(m_run[i] - m_all);
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][2 * i] *= f;
          o[n][2 * i + 1] *= f;
        }
        if (warp == 0 && tq == 0) {
          red_m[C::kWarps * 16 + g + 8 * i] = m_all;
          red_l[C::kWarps * 16 + g + 8 * i] = l_all;
        }
      }
      auto stage = [&](int at, bool add) {
        float* const dst = merge + at * 16 * D;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float2* const x = reinterpret_cast<float2*>(dst + (g + 8 * i) * D + n * 8 + 2 * tq);
            float2 y = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            if (add) {
              const float2 z = *x;
              y.x += z.x;
              y.y += z.y;
            }
            *x = y;
          }
      };
      constexpr int kHalf = C::kWarps / 2;
      if (warp >= kHalf) stage(warp - kHalf, false);
      __syncthreads();
      if (warp < kHalf) stage(warp, true);
      __syncthreads();
      if constexpr (kHalf == 2) {
        for (int i = threadIdx.x; i < 16 * D / 4; i += C::kThreads) {
          float4* const x = reinterpret_cast<float4*>(merge) + i;
          const float4 y = *x, z = reinterpret_cast<const float4*>(merge + 16 * D)[i];
          *x = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
        }
        __syncthreads();
      }
      put_unit<T, D, RU, SR, C::kThreads>(a, wc, whole, red_m + C::kWarps * 16, red_l + C::kWarps * 16, merge);
      __syncthreads();
    }
    if (s + 1 < total) wc.next(a);
  }
  cp_async_wait<0>();
  end_main(a);
}

// ---- fp32 caches --------------------------------------------------------------------

template <int D, int kRows>
struct PagedF32 {
  static constexpr int RU = kRows;
  static constexpr int kThreads = 128;
  static constexpr int SR = D == 256 ? 16 : 32;
  static constexpr int kParts = kThreads / SR;       // lanes that share out a key's row
  static constexpr int kVec = D / 4;                 // columns of the second product, four at a time
  static constexpr int kSlices = kThreads / kVec;    // threads that share out a column's keys
  static constexpr int kStageBytes = SR * D * 4;     // per tensor
  static constexpr int kStages = 96 * 1024 / (2 * kStageBytes) < 6 ? 96 * 1024 / (2 * kStageBytes) : 6;
  static constexpr int kOffQ = 2 * kStages * kStageBytes;
  static constexpr int kOffP = kOffQ + RU * D * 4;
  static constexpr int kOffMl = kOffP + RU * SR * 4;
  static constexpr int kOffMerge = kOffMl + 4 * RU * 4;
  static constexpr int kOffOk = kOffMerge + RU * D * 4;
  static constexpr int kSmemBytes = kOffOk + kStages * (SR / 16) * 4;
};

template <int D, int kRows>
__global__ void __launch_bounds__(128) paged_f32_kernel(PagedArgs a) {
  using C = PagedF32<D, kRows>;
  constexpr int SR = C::SR, RU = C::RU, kStages = C::kStages, kThreads = C::kThreads;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const k_ring = smem;
  unsigned char* const v_ring = smem + kStages * C::kStageBytes;
  float* const q_s = reinterpret_cast<float*>(smem + C::kOffQ);        // [row][D], times scale
  float* const p_s = reinterpret_cast<float*>(smem + C::kOffP);        // [key][row]
  float* const m_s = reinterpret_cast<float*>(smem + C::kOffMl);       // running (m, l) and the stage's factor of every row
  float* const l_s = m_s + RU;
  float* const f_s = l_s + RU;
  float* const merge = reinterpret_cast<float*>(smem + C::kOffMerge);  // [row][D]
  int* const ok_ring = reinterpret_cast<int*>(smem + C::kOffOk);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  begin_main(a);
  Walk<SR> wc;
  long long per;
  const int total = find_share<SR, kThreads>(a, &wc, &per);
  if (total == 0) {
    end_main(a);
    return;
  }
  Walk<SR> wi = wc;
  Loader<float, D, SR, kThreads> load;
  load.look_up(a, wi);
  int issued = 0;
  auto issue = [&]() {
    if (issued < total) {
      const int slot = issued % kStages;
      load.issue(a, wi, k_ring + slot * C::kStageBytes, v_ring + slot * C::kStageBytes, ok_ring + slot * (SR / 16));
      if (++issued < total) {
        wi.next(a);
        load.look_up(a, wi);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue();

  const int key = tid / C::kParts, part = tid % C::kParts;         // first product
  const int col = tid % C::kVec, slice = tid / C::kVec;            // second product
  float4 o[RU];
  int first_st = wc.st;
  for (int s = 0; s < total; ++s) {
    if (s == 0 || wc.st == 0) {
      first_st = wc.st;
      for (int i = tid; i < RU * C::kVec; i += kThreads) {
        int b, h;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (unit_row<RU>(a, wc, i / C::kVec, &b, &h))
          x = reinterpret_cast<const float4*>(a.q)[(static_cast<size_t>(b) * a.H + h) * C::kVec + i % C::kVec];
        reinterpret_cast<float4*>(q_s)[i] = x;
      }
      if (tid < RU) {
        m_s[tid] = -INFINITY;
        l_s[tid] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < RU; ++r) o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    cp_async_wait<kStages - 2>();
    __syncthreads();
    issue();
    const int slot = s % kStages;
    const int n_valid = wc.end - wc.start - wc.st * SR;
    // scores: kParts lanes a key, every kParts-th piece each
    {
      const float4* const row = reinterpret_cast<const float4*>(k_ring + slot * C::kStageBytes) + key * C::kVec;
      float sc[RU];
#pragma unroll
      for (int r = 0; r < RU; ++r) sc[r] = 0.f;
#pragma unroll 4
      for (int j = 0; j < C::kVec / C::kParts; ++j) {
        const int c = j * C::kParts + part;
        const float4 x = row[load.place(key, c)];
#pragma unroll
        for (int r = 0; r < RU; ++r) {
          const float4 y = reinterpret_cast<const float4*>(q_s)[r * C::kVec + c];
          sc[r] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, sc[r]))));
        }
      }
      const bool seen = key < n_valid && ok_ring[slot * (SR / 16) + (key >> 4)];
#pragma unroll
      for (int r = 0; r < RU; ++r) {
#pragma unroll
        for (int i = 1; i < C::kParts; i *= 2) sc[r] += __shfl_xor_sync(0xffffffffu, sc[r], i);
        if (part == r % C::kParts) p_s[key * RU + r] = seen ? sc[r] * a.scale_log2 : -INFINITY;
      }
    }
    __syncthreads();
    // a warp a row: maximum, weights, sum
    for (int r = warp; r < RU; r += 4) {
      const float v = lane < SR ? p_s[lane * RU + r] : -INFINITY;
      float mx = v;
#pragma unroll
      for (int i = 16; i > 0; i /= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
      const float m_old = m_s[r], m_new = fmaxf(m_old, mx);
      const float p = ex2(v - (m_new == -INFINITY ? 0.f : m_new));
      float sum = p;
#pragma unroll
      for (int i = 16; i > 0; i /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, i);
      if (lane < SR) p_s[lane * RU + r] = p;
      __syncwarp();
      if (lane == 0) {
        const float f = m_old == -INFINITY ? (l_s[r] == 0.f ? 0.f : 1.f) : ex2(m_old - m_new);
        f_s[r] = f;
        l_s[r] = l_s[r] * f + sum;
        m_s[r] = m_new;
      }
    }
    __syncthreads();
    // values: a thread has four columns and every kSlices-th key
    {
      const float4* const v_s = reinterpret_cast<const float4*>(v_ring + slot * C::kStageBytes);
#pragma unroll
      for (int r = 0; r < RU; ++r) {
        const float f = f_s[r];
        o[r].x *= f;
        o[r].y *= f;
        o[r].z *= f;
        o[r].w *= f;
      }
      const int* const ok = ok_ring + slot * (SR / 16);
#pragma unroll 4
      for (int i = 0; i < SR / C::kSlices; ++i) {
        const int j = i * C::kSlices + slice;
        if (j >= n_valid || !ok[j >> 4]) continue;
        const float4 x = v_s[j * C::kVec + load.place(j, col)];
#pragma unroll
        for (int r = 0; r < RU; ++r) {
          const float p = p_s[j * RU + r];
          o[r].x = fmaf(p, x.x, o[r].x);
          o[r].y = fmaf(p, x.y, o[r].y);
          o[r].z = fmaf(p, x.z, o[r].z);
          o[r].w = fmaf(p, x.w, o[r].w);
        }
      }
    }
    if (wc.st == wc.n - 1 || s == total - 1) {
      const bool whole = first_st == 0 && wc.st == wc.n - 1;
      // the slices of a column one after the other
      for (int i = 0; i < C::kSlices; ++i) {
        if (slice == i) {
#pragma unroll
          for (int r = 0; r < RU; ++r) {
            float4* const x = reinterpret_cast<float4*>(merge) + r * C::kVec + col;
            const float4 y = i == 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *x;
            *x = make_float4(y.x + o[r].x, y.y + o[r].y, y.z + o[r].z, y.w + o[r].w);
          }
        }
        __syncthreads();
      }
      put_unit<float, D, RU, SR, kThreads>(a, wc, whole, m_s, l_s, merge);
      __syncthreads();
    }
    if (s + 1 < total) wc.next(a);
  }
  cp_async_wait<0>();
  end_main(a);
}

// ---- fold ---------------------------------------------------------------------------

// Parts of the rows that no block finished. A row has D / 4 threads, four columns each, times kSlices, which take every
// kSlices-th part.
constexpr int kFoldThreads = 256;
template <typename T, int D, int SR, int RU, int kSlices>
__global__ void __launch_bounds__(kFoldThreads) paged_fold_kernel(const PagedArgs a) {
  constexpr int kVec = D / 4, kRowsPer = kFoldThreads / kVec / kSlices;
  __shared__ float4 acc_of[kSlices > 1 ? kFoldThreads : 1];
  __shared__ float2 ml_of[kSlices > 1 ? kFoldThreads / kVec : 1];
  let_next_start();
  const int col = threadIdx.x % kVec, lane_row = threadIdx.x / kVec, slice = lane_row % kSlices;
  const int row = static_cast<int>(blockIdx.x) * kRowsPer + lane_row / kSlices;
  const bool mine = row < a.B * a.H;
  const int b = mine ? row / a.H : 0, h = mine ? row - b * a.H : 0, kvh = h % a.kvH, g = h / a.kvH;
  wait_for_previous();
  int start = 0, end = 0;
  if (mine) own_keys(a, b, &start, &end);
  const int n = static_cast<int>((static_cast<long long>(end) - start + SR - 1) / SR);
  const long long per = a.head[0];
  // parts [lo, lo + count) of a unit: those of the blocks that its stages lie with
  long long own_lo = 0, pre_lo = 0;
  int own_n = 0, pre_n = 0;
  if (mine && n > 0) {
    const int hb = g / RU;
    const long long beg = a.head[1 + b] + static_cast<long long>(kvh * a.HB + hb) * n;
    const long long c0 = beg / per, c1 = (beg + n - 1) / per;
    const long long uid = static_cast<long long>(a.kvH) * a.RB + (static_cast<long long>(b) * a.kvH + kvh) * a.HB + hb;
    own_lo = (c0 + uid) * a.rs + g % RU;
    own_n = static_cast<int>(c1 - c0) + 1;
  }
  if (mine && start > 0 && a.RB > 0) {
    const int i = b * a.G + g, tile = i / RU, stages = (a.shared_len + SR - 1) / SR;
    const long long uid = static_cast<long long>(kvh) * a.RB + tile, beg = uid * stages;
    const long long c0 = beg / per, c1 = (beg + stages - 1) / per;
    pre_lo = (c0 + uid) * a.rs + i % RU;
    pre_n = static_cast<int>(c1 - c0) + 1;
  }
  long long pre_step = a.rs;
  const float2* pre_ml = a.part_ml;
  const float* pre_o = a.part_o;
  bool lost = false;  // the kernel of the shared pages gave up: the rows stay as they are
  if (a.shared_ml) {
    lost = *reinterpret_cast<const volatile int*>(a.status) != 0;
    if (mine && start > 0) {
      const SharedPlan& s = a.shared;
      const int tile = s.pack > 1 ? g / s.pack : b / 128 * a.G + g, at = s.pack > 1 ? g % s.pack * a.B + b : b % 128;
      pre_step = s.tiles_per_block * 128;
      pre_lo = (static_cast<long long>(kvh) * s.blocks + tile / s.tiles_per_block) * s.shares * pre_step +
               tile % s.tiles_per_block * 128 + at;
      pre_n = s.shares;
      pre_ml = a.shared_ml;
      pre_o = a.shared_o;
    }
  }
  const bool done = lost || (own_n == 1 && start == 0);  // by the block that had the unit
  const int parts = mine && !done ? own_n + pre_n : 0;
  auto ml_of_part = [&](int i) { return i < pre_n ? pre_ml[pre_lo + i * pre_step] : a.part_ml[own_lo + static_cast<long long>(i - pre_n) * a.rs]; };
  auto o_of_part = [&](int i) {
    const float* const o = i < pre_n ? pre_o + (pre_lo + i * pre_step) * D : a.part_o + (own_lo + static_cast<long long>(i - pre_n) * a.rs) * D;
    return *reinterpret_cast<const float4*>(o + col * 4);
  };
  float m_all = -INFINITY;
#pragma unroll 4
  for (int i = slice; i < parts; i += kSlices) m_all = fmaxf(m_all, ml_of_part(i).x);
  float l_all = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = slice; i < parts; i += kSlices) {
    const float2 ml = ml_of_part(i);
    const float4 o = o_of_part(i);
    if (ml.y == 0.f) continue;  // saw nothing
    const float f = ml.x > -INFINITY ? ex2(ml.x - m_all) : 1.f;
    l_all += f * ml.y;
    acc.x += f * o.x;
    acc.y += f * o.y;
    acc.z += f * o.z;
    acc.w += f * o.w;
  }
  if constexpr (kSlices > 1) {
    acc_of[threadIdx.x] = acc;
    if (col == 0) ml_of[lane_row] = make_float2(m_all, l_all);
    __syncthreads();
    if (slice == 0) {
      const float2 own = make_float2(m_all, l_all);
#pragma unroll
      for (int i = 1; i < kSlices; ++i) m_all = fmaxf(m_all, ml_of[lane_row + i].x);
      const float f0 = own.x > -INFINITY ? ex2(own.x - m_all) : 1.f;
      l_all = f0 * own.y;
      acc = make_float4(f0 * acc.x, f0 * acc.y, f0 * acc.z, f0 * acc.w);
#pragma unroll
      for (int i = 1; i < kSlices; ++i) {
        const float2 ml = ml_of[lane_row + i];
        const float4 o = acc_of[threadIdx.x + i * kVec];
        const float f = ml.x > -INFINITY ? ex2(ml.x - m_all) : 1.f;
        l_all += f * ml.y;
        acc.x += f * o.x;
        acc.y += f * o.y;
        acc.z += f * o.z;
        acc.w += f * o.w;
      }
    }
  }
  if (!mine || done || slice != 0) return;
  const bool any = l_all != 0.f;  // (NaN counts)
  const float inv = 1.f / l_all;
  put4(static_cast<T*>(a.out) + static_cast<size_t>(row) * D + col * 4,
       any ? make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f));
  if (a.lse && col == 0) a.lse[row] = l_all > 0.f ? m_all * kLn2 + logf(l_all) : any ? l_all : -INFINITY;
}

// ---- host side ----------------------------------------------------------------------

// Which kernel a call runs, and its room: header, (m, l) and O of every part. A block leaves at most one part a unit, and
// block c's of unit u is part c + u: both only grow along the list, so no two meet.
struct PagedPlan {
  int RU, SR, blocks;
  bool tc;  // shared pages by the tensor-core kernel
  SharedPlan shared;
  double most;  // stages that there can be
  int rs;  // rows of a part
  size_t parts, head_bytes, ml_bytes, o_bytes, shared_rows, shared_ml_bytes, bytes;
};

constexpr int kBlocksPerSm = 2;  // of both kernels: 96 KB of ring each

int fp32_rows(int G) { return G <= 1 ? 1 : G <= 2 ? 2 : G <= 4 ? 4 : 8; }

PagedPlan make_plan(const ra_paged_kv& c, int heads, int shared_len) {
  PagedPlan p = {};
  const int G = (heads + c.kv_heads - 1) / c.kv_heads;
  const bool f32 = c.dtype == RA_F32;
  const long long rows_shared = shared_len > 0 ? static_cast<long long>(c.batch) * G : 0;
  p.RU = f32 ? fp32_rows(static_cast<int>(std::max<long long>(std::min<long long>(rows_shared, 8), G))) : 16;
  p.SR = f32 ? (c.head_dim == 256 ? 16 : 32) : c.head_dim == 256 ? 32 : 64;
  p.tc = !f32 && rows_shared > 0 && static_cast<long long>(c.num_pages) * c.kv_heads < (1ll << 31) - 1 && c.num_pages > 0 &&
         plan_shared_prefix(c.batch, heads, c.kv_heads, c.head_dim, shared_len, &p.shared);
  const long long HB = (G + p.RU - 1) / p.RU, RB = p.tc ? 0 : (rows_shared + p.RU - 1) / p.RU;
  const long long units = c.kv_heads * (RB + c.batch * HB);
  // stages that there are at most: as many as the tables have room for
  const long long room = static_cast<long long>(c.max_pages) * c.page_size;
  p.most = static_cast<double>(c.kv_heads) * (static_cast<double>(c.batch) * HB * ((room + p.SR - 1) / p.SR) +
                                                   static_cast<double>(RB) * ((shared_len + p.SR - 1) / p.SR));
  const int wave = kBlocksPerSm * sm_count();
  p.blocks = p.most < wave ? static_cast<int>(p.most) : wave;
  p.parts = static_cast<size_t>(units) + p.blocks;
  p.rs = RB > 0 ? p.RU : std::min(p.RU, G);
  const size_t rs = p.rs;
  auto whole = [](size_t n) { return (n + 127) & ~static_cast<size_t>(127); };
  p.head_bytes = whole((1 + static_cast<size_t>(c.batch)) * 8);
  p.ml_bytes = whole(p.parts * rs * sizeof(float2));
  p.o_bytes = whole(p.parts * rs * c.head_dim * sizeof(float));
  p.shared_rows = p.tc ? shared_part_rows(p.shared, c.kv_heads) : 0;
  p.shared_ml_bytes = whole(p.shared_rows * sizeof(float2));
  p.bytes = p.head_bytes + p.ml_bytes + p.o_bytes + p.shared_ml_bytes + p.shared_rows * c.head_dim * sizeof(float);
  return p;
}

template <void (*kern)(PagedArgs)>
int launch_main(int threads, int smem, int blocks, const PagedArgs& a, cudaStream_t stream) {
  static std::atomic<unsigned long long> smem_set{0};  // once per device and instantiation
  int dev = 0;
  RAB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !(smem_set.load(std::memory_order_acquire) >> dev & 1ull)) {
    RAB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev >= 0 && dev < 64) smem_set.fetch_or(1ull << dev, std::memory_order_release);
  }
  RAB_CUDA(launch_overlapped(kern, dim3(static_cast<unsigned>(blocks)), dim3(threads), smem, stream, a));
  return RA_OK;
}

template <typename T, int D, int SR, int RU>
int launch_fold(const PagedArgs& a, int blocks, cudaStream_t stream) {
  const long long rows = static_cast<long long>(a.B) * a.H;
  constexpr int kPer = kFoldThreads / (D / 4);
  if (rows * 4 <= blocks) {
    RAB_CUDA(launch_overlapped(paged_fold_kernel<T, D, SR, RU, 4>, dim3(static_cast<unsigned>((rows + kPer / 4 - 1) / (kPer / 4))),
                               dim3(kFoldThreads), 0, stream, a));
  } else {
    RAB_CUDA(launch_overlapped(paged_fold_kernel<T, D, SR, RU, 1>, dim3(static_cast<unsigned>((rows + kPer - 1) / kPer)),
                               dim3(kFoldThreads), 0, stream, a));
  }
  return RA_OK;
}

template <typename T, int D>
int launch_16(const PagedArgs& a, const PagedPlan& p, cudaStream_t stream) {
  using C = PagedMma<D>;
  if (p.blocks > 0) {
    const int rc = launch_main<paged_mma_kernel<T, D>>(C::kThreads, C::kSmemBytes, p.blocks, a, stream);
    if (rc != RA_OK) return rc;
  }
  return launch_fold<T, D, C::SR, C::RU>(a, p.blocks, stream);
}

template <int D, int RU>
int launch_32(const PagedArgs& a, const PagedPlan& p, cudaStream_t stream) {
  using C = PagedF32<D, RU>;
  if (p.blocks > 0) {
    const int rc = launch_main<paged_f32_kernel<D, RU>>(C::kThreads, C::kSmemBytes, p.blocks, a, stream);
    if (rc != RA_OK) return rc;
  }
  return launch_fold<float, D, C::SR, RU>(a, p.blocks, stream);
}

template <int D>
int launch_head_dim(int dtype, const PagedArgs& a, const PagedPlan& p, cudaStream_t stream) {
  if (dtype == RA_F16) return launch_16<__half, D>(a, p, stream);
  if (dtype == RA_BF16) return launch_16<__nv_bfloat16, D>(a, p, stream);
  if (p.RU == 1) return launch_32<D, 1>(a, p, stream);
  if (p.RU == 2) return launch_32<D, 2>(a, p, stream);
  if (p.RU == 4) return launch_32<D, 4>(a, p, stream);
  return launch_32<D, 8>(a, p, stream);
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
  RAB_REQUIRE(shared_len >= 0 && shared_len % c.page_size == 0 && (shared_len == 0 || shared_pages), RA_ERR_INVALID,
              "%s: shared pages are whole: shared_len=%d, page_size=%d", what, shared_len, c.page_size);
  return RA_OK;
}

}  // namespace
}  // namespace rab

using namespace rab;

extern "C" {

size_t ra_paged_decode_workspace_bytes(const ra_paged_kv* cache, int heads, int shared_len) {
  if (!cache) return 0;
  ra_paged_kv c = *cache;
  int none = 0;
  if (check_decode(c, heads, &none, shared_len) != RA_OK) return 0;
  return make_plan(c, heads, shared_len).bytes;
}

int ra_paged_decode(const ra_paged_kv* cache, const void* q, int heads, const int* shared_pages, int shared_len, void* out,
                    float* lse, void* workspace, size_t workspace_bytes, ra_stream stream_) {
  RAB_REQUIRE(cache != nullptr, RA_ERR_INVALID, "paged_decode: null argument");
  const ra_paged_kv& c = *cache;
  const int rc = check_decode(c, heads, shared_pages, shared_len);
  if (rc != RA_OK) return rc;
  if (c.batch == 0) return RA_OK;
  RAB_REQUIRE(q && out, RA_ERR_INVALID, "paged_decode: null argument");
  RAB_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0, RA_ERR_INVALID,
              "paged_decode: q and out must be 16-byte aligned");
  const PagedPlan p = make_plan(c, heads, shared_len);
  // (a share is counted in 32 bits; tables that name a page over and over could ask for more)
  RAB_REQUIRE(p.most < 2147483648.0 * std::max(p.blocks, 1), RA_ERR_INVALID, "paged_decode: too many keys");
  RAB_REQUIRE(workspace && workspace_bytes >= p.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, RA_ERR_OVERFLOW,
              "paged_decode: workspace too small or not 16-byte aligned");
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
  a.shared_len = shared_len;
  a.num_pages = c.num_pages;
  a.max_pages = c.max_pages;
  a.shift = page_shift(c.page_size);
  a.B = c.batch;
  a.H = heads;
  a.kvH = c.kv_heads;
  a.G = (heads + c.kv_heads - 1) / c.kv_heads;
  a.HB = (a.G + p.RU - 1) / p.RU;
  a.RB = shared_len > 0 && !p.tc ? static_cast<int>((static_cast<long long>(a.B) * a.G + p.RU - 1) / p.RU) : 0;
  a.rs = p.rs;
  a.min_per = 1;
  a.scale_log2 = kLog2e / std::sqrt(static_cast<float>(c.head_dim));
  unsigned char* const ws = static_cast<unsigned char*>(workspace);
  a.head = reinterpret_cast<long long*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + p.head_bytes);
  a.part_o = reinterpret_cast<float*>(ws + p.head_bytes + p.ml_bytes);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  a.shared = p.shared;
  a.shared_ml = nullptr;
  a.shared_o = nullptr;
  a.status = nullptr;
  if (p.tc) {
    a.shared_ml = reinterpret_cast<float2*>(ws + p.head_bytes + p.ml_bytes + p.o_bytes);
    a.shared_o = reinterpret_cast<float*>(ws + p.head_bytes + p.ml_bytes + p.o_bytes + p.shared_ml_bytes);
    a.status = device_status_ptr();
    const SharedPrefix s{q, c.k, c.v, a.B, a.H, a.kvH, c.head_dim, shared_pages, c.lens, shared_len, c.num_pages, c.max_pages, a.shift};
    const int rc2 = launch_shared_prefix(c.dtype, s, p.shared, a.shared_o, a.shared_ml, stream);
    if (rc2 != RA_OK) return rc2;
  }
  if (c.head_dim == 32) return launch_head_dim<32>(c.dtype, a, p, stream);
  if (c.head_dim == 64) return launch_head_dim<64>(c.dtype, a, p, stream);
  if (c.head_dim == 128) return launch_head_dim<128>(c.dtype, a, p, stream);
  return launch_head_dim<256>(c.dtype, a, p, stream);
}

}  // extern "C"
