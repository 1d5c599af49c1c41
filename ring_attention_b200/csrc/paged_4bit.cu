// Decode attention (one query row a sequence) against a paged KV cache whose rows are held in 4 bits, and rows of a paged cache
// of any kind read back out of it.
//
// A row x of K or V is held as 16 elements to a block: a scale s in e4m3 (3 bits of fraction, up to 448), and for each element a
// code c in e2m1, one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign; the element's value is c s f, f a power of two for the whole of K or
// of V. c s has at most 5 significant bits, so it is exact in fp16 (2^-10 to 2688) and the products below see the cached values as
// they are. A row is 9/16 of its elements' number in bytes.
//
//   out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(q . k_j / sqrt(D)),  j < lens[b],  KV head h % kv_heads
//
// The walk is that of paged_decode.cu (paged_walk.cuh). What is different is that a byte of the cache brings two elements and so four
// times the instructions of a 16-bit one: besides the copy the issue slots bound it. So nothing is moved for the tensor core's sake: both
// products have the cached operand as the A of mma.sync m16n8k16 (16 keys by 16 columns of K, 16 columns by 16 keys of V), eight
// query heads as its N, and each lane makes its part of A in registers from the bytes of its own rows: the order of the columns
// in a contraction is free, so a lane takes 16 columns of K that lie side by side, and 16 of V. A code pair becomes two fp16 by one
// conversion and their scales one multiplication.
//
// What bounds it: 290 warp instructions to 16 keys of 128 columns (116 of them V's, 82 K's), of which the conversions, V's change of places
// and the scores' comparisons, 130, are the ALU pipe's at half rate: 59 % of the issue slots, three warps a scheduler. Without copies, 64
// sequences of up to 8191 rows (H32/kvH8 D128, 454 MB) took 92 us, the copies alone 77.
//
// Measured, us in a CUDA graph, and the floor of the cache's bytes at the copy's rate:
//
//   64 sequences of up to 8191 rows, H32/kvH8 D128         111   69
//   64 sequences of 4096 to 8191, H32/kvH8 D32, 64, 128    53, 71, 104   17, 35, 69 (the instructions of a row are nearly as many)
//   4 sequences of up to 262144 rows, H32/kvH8 D128        202   145 (the same rows in 16 bits: 502)
//   5 sequences of up to 33333 rows, H32/kvH2 D256         50    11.5 (16 heads: 255 registers, two warps a scheduler, 102 bytes spilled)
//
// Eight warps a block with copies of 32 keys instead of six with 64: 114 and 216 us for the first and the third.
#include "paged_walk.cuh"

namespace rab {

namespace {

// ---- decode -------------------------------------------------------------------------

struct FourArgs {
  PagedArgs p;
  float k_factor, v_factor;
};

// The list of stages is one of kGrain keys each, so that short calls divide over all warps; a copy takes as many of them, up to GR, as a
// share has left of a unit, because what surrounds a copy costs some 300 instructions and 16 keys of 128 columns 280.
constexpr int kGrain = 32;
constexpr int four_warps(int D, int NB) { return D * NB <= 128 ? 6 : 4; }  // of a block

template <int D, int NB>
struct FourBlock {
  static constexpr int GR = D >= 256 ? 1 : D == 128 ? 2 : 4, SR = GR * kGrain, RU = 8 * NB;
  // accumulators and queries: (D / 4 + D / 8) NB registers
  static constexpr int kWarps = four_warps(D, NB), kThreads = kWarps * 32;
  static constexpr int kCodeBytes = D / 2, kScaleBytes = D / 16, kRowBytes = kCodeBytes + kScaleBytes;
  static constexpr int kTileBytes = SR * kRowBytes;  // per tensor: codes, then scales
  static constexpr int kMost = 110 * 1024 / kWarps / (2 * kTileBytes);
  static constexpr int kStages = kMost < 4 ? kMost : 4;
  static constexpr int kRingBytes = 2 * kStages * kTileBytes;
  static constexpr int kOffInfo = kWarps * kRingBytes;
  static constexpr int kOffUnits = kOffInfo + ((kWarps * kStages * 4 + 15) & ~15);
  static constexpr int kOffBar = kOffUnits + kWarps * kStages * 16;
  static constexpr int kOffRoom = (kOffBar + kWarps * kStages * 8 + 15) & ~15;
  static constexpr int kOffFlag = kOffRoom + static_cast<int>(sizeof(ScanRoom<kWarps>));
  static constexpr int kSmemBytes = kOffFlag + 8;
  static_assert(kTileBytes % 16 == 0 && kStages >= 2, "the ring");
  static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two blocks to an SM");
};

// The reference of the weights is moved only when a score runs kSlack above it (in log2): with sixteen heads some maximum moves in nearly
// every one of a share's first tiles, at 200 instructions each time. The reference's own weight is 2^kLift, because what is 2^-25 and less
// is 0 in fp16 while it counts in the weights' sum: so those below 2^-32 of the reference's do, not those below 2^-25 (of 300000 keys
// that may be 1 %). Together 2^14 at most, and 2^15 where the reference less kLift is rounded: fp16 goes up to 2^16.
constexpr float kSlack = 7.f, kLift = 7.f;

// A warp's ring: while a place is worked on, the others' copies are on their way.
template <typename C>
struct FourRing {
  const PagedArgs& a;
  unsigned char* tiles;  // shared memory: the ring, what there is to know of its places (see Info), the units of their keys, barriers
  unsigned* info;
  int4* units;
  unsigned full;
  volatile int* gave_up;
  Walk<kGrain> w;  // the unit whose grains are copied
  int total, per, next;
  // of the warp's part of that unit: grains that are left, keys of the unit that are, the next key, whether nothing is copied yet
  int run, left, at;
  bool fresh, whole;  // (whole: the part is all of the unit)
  const int* table;
  // this lane's copies: piece `piece` of the rows, of K's or V's codes or scales
  const unsigned char* from;
  unsigned to, row_bytes, rows, offset;
  int kind, page;  // (page: of its next copy, -1: none)

  // What a warp has to know of a place when its copy has landed: keys (8 bits), blocks of 16 keys that are there (8), first of its part of
  // the unit (1), last of it (1: yes, 2: yes, and the part is the result).
  static constexpr int kBlocks = 8, kFirst = 16, kLast = 17;

  __device__ inline void begin_part() {
    run = min(w.n - w.st, total - next);
    left = w.left();
    at = w.st * kGrain;
    fresh = true;
    whole = w.st == 0 && run == w.n;
    table = a.table + w.b * a.table_stride;
    // the warp with a unit's first grain says which shares have parts of it: its own and those that the rest reaches into
    if (w.st == 0 && (threadIdx.x & 31) == 0)
      a.unit_parts[w.uid] = make_int2(static_cast<int>(blockIdx.x * C::kWarps + (threadIdx.x >> 5)), 1 + (w.n - run + per - 1) / per);
  }
  __device__ inline void look_up() {  // (the keys of a unit lie in its table)
    page = run > 0 && kind < 4 && static_cast<int>(offset) < left ? table[(at + static_cast<int>(offset)) >> a.shift] : -1;
  }
  __device__ inline void begin(unsigned base) {
    const unsigned lane = threadIdx.x & 31, shift = a.shift < 5 ? a.shift : 5, pieces = C::SR >> shift;
    rows = 1u << shift;
    offset = lane % pieces * rows;
    kind = lane / pieces;
    const int which = kind >> 1;  // 0: codes, 1: scales
    row_bytes = which == 0 ? C::kCodeBytes : C::kScaleBytes;
    from = static_cast<const unsigned char*>((kind & 1) == 0 ? a.k : a.v) + (which == 0 ? 0 : C::kCodeBytes << a.shift);
    to = base + (kind & 1) * C::kTileBytes + (which == 0 ? 0 : C::SR * C::kCodeBytes) + offset * row_bytes;
    next = 0;
    begin_part();
    look_up();
    for (int s = 0; s < C::kStages; ++s) copy(s);
  }
  // Copies the next grains, if there are any, to a place that is free.
  __device__ inline void copy(int slot) {
    if (run == 0) return;
    const int grains = min(C::GR, run), keys = min(grains * kGrain, left);
    const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages) && static_cast<int>(offset) < keys;
    const unsigned pieces = __ballot_sync(0xffffffffu, there && kind == 0);
    if ((threadIdx.x & 31) == 0) {
      unsigned blocks = pieces;
      if (rows == 32) blocks = (pieces & 1u) * 3u | (pieces & 2u) * 6u | (pieces & 4u) * 12u | (pieces & 8u) * 24u;
      info[slot] = static_cast<unsigned>(keys) | blocks << kBlocks | static_cast<unsigned>(fresh) << kFirst |
                   (run > grains ? 0u : whole ? 2u : 1u) << kLast;
      if (fresh) units[slot] = make_int4(w.b, w.kvh, w.hb, w.uid);
      tcgen::mbar_expect_tx(full + 8 * slot, 2 * C::kRowBytes * rows * __popc(pieces) + a.missing);
    }
    __syncwarp();
    if (there) {
      const int row = (at + static_cast<int>(offset)) & ((1 << a.shift) - 1);
      tcgen::bulk_load(to + 2 * slot * C::kTileBytes,
                       from + ((static_cast<size_t>(page) * a.kvH + w.kvh) << a.shift) * C::kRowBytes + row * row_bytes, row_bytes * rows,
                       full + 8 * slot);
    }
    fresh = false;
    at += grains * kGrain;
    left -= grains * kGrain;
    next += grains;
    run -= grains;
    if (run == 0 && next < total) {  // on to the next unit
      w.st = w.n - 1;
      w.next(a);
      begin_part();
    }
    look_up();
  }
  // Waits for copy s; false: the warp gives up.
  __device__ inline bool wait(int s) {
    return __all_sync(0xffffffffu, tcgen::mbar_wait(full + 8 * (s % C::kStages), (s / C::kStages) & 1, gave_up, a.status, 3, s,
                                                    a.wait_ns)) != 0;
  }
};

// The eight codes of a word as fp16 pairs, neighbours together.
__device__ inline void codes_to_half(unsigned w, unsigned (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// Two scales as fp16.
__device__ inline unsigned scales_to_half(unsigned short s) {
  unsigned h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(s));
  return h;
}
__device__ inline unsigned mul_half2(unsigned a, unsigned b) {
  unsigned d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// An 8 x 8 matrix of 16-bit elements over the warp, transposed.
__device__ inline unsigned transposed(unsigned a) {
  unsigned d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Words of shared memory, N of them.
template <int N>
__device__ inline void load_words(const unsigned char* p, unsigned (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const unsigned*>(p);
  }
}
__device__ inline unsigned load_u16(const unsigned char* p) { return *reinterpret_cast<const unsigned short*>(p); }

// Where the products' places are. Lane (g, j) of a fragment has its rows g and g + 8 and its columns 2 j, 2 j + 1, 2 j + 8, 2 j + 9.
// Key at place p of 16: p ^ (p >> 2 & 1), so that the keys 2 j differ in the rest by four, as do the keys g of half a warp: with the
// pieces' places in a page (four_turn) no two lanes of an access meet in a bank.
// K: columns of step s, lane j: from k_column on, two and two. V: columns of tile i, lane g: v_column of its row g, and v_other
// behind it that of its row g + 8.
__device__ inline int key_at(int place) { return place ^ (place >> 2 & 1); }
template <int D>
struct FourCols {
  static constexpr int kRun = D >= 128 ? 32 : D / 4;  // columns of K that a lane has side by side
  static constexpr int kVCols = D / 8;                // of V
  static constexpr int v_other = D / 16;
  __device__ static int k_column(int s, int j) { return D >= 128 ? s / 8 * 128 + 32 * j + s % 8 * 4 : kRun * j + 4 * s; }
  __device__ static int v_column(int i, int g) { return kVCols * g + i; }
};

template <typename T, int D, int NB>
__global__ void __launch_bounds__(FourBlock<D, NB>::kThreads, 2) paged_4bit_kernel(const __grid_constant__ FourArgs args) {
  using C = FourBlock<D, NB>;
  using Cols = FourCols<D>;
  constexpr int RU = C::RU, kSteps = D / 16, kTiles = D / 16;
  constexpr int kT = D * NB <= 256 ? 2 : 1;  // tiles of 16 keys at a time: two, as far as the registers go
  extern __shared__ __align__(1024) unsigned char smem[];
  const PagedArgs& a = args.p;
  const unsigned base = tcgen::smem_u32(smem);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  volatile int* const gave_up = reinterpret_cast<volatile int*>(smem + C::kOffFlag);
  let_next_start();
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kWarps * C::kStages; ++s) tcgen::mbar_init(base + C::kOffBar + 8 * s, 1);
    *gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  wait_for_previous();
  FourRing<C> ring{a, smem + warp * C::kRingBytes, reinterpret_cast<unsigned*>(smem + C::kOffInfo) + warp * C::kStages,
                   reinterpret_cast<int4*>(smem + C::kOffUnits) + warp * C::kStages, base + C::kOffBar + warp * C::kStages * 8, gave_up};
  ring.total = find_share<kGrain, C::kWarps>(a, warp, &ring.w, &ring.per, reinterpret_cast<ScanRoom<C::kWarps>*>(smem + C::kOffRoom));
  auto walk = [&]() {
    ring.begin(base + warp * C::kRingBytes);
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    const int key_g = key_at(g), key_0 = key_at(2 * j), key_1 = key_at(2 * j + 1);
    const int turn_g = four_turn(key_g, D), turn_0 = four_turn(key_0, D), turn_1 = four_turn(key_1, D);
    constexpr int kKWords = Cols::kRun / 8, kKPieces = D == 256 ? 2 : 1;
    constexpr int kVWords = D >= 64 ? D / 64 : 1;
    // offsets of a lane's bytes in a tile of 16 keys, codes and scales (the turn of a key and of the key 8 behind it are the same)
    unsigned k_at[kKPieces], v_at[2];
#pragma unroll
    for (int p = 0; p < kKPieces; ++p)
      k_at[p] = key_g * C::kCodeBytes + (D >= 128 ? ((j + 4 * p) ^ turn_g) * 16 : j * (D / 8));
    const int v_byte = g * (D / 16);
    v_at[0] = key_0 * C::kCodeBytes + ((v_byte / 16) ^ turn_0) * 16 + v_byte % 16;
    v_at[1] = key_1 * C::kCodeBytes + ((v_byte / 16) ^ turn_1) * 16 + v_byte % 16;
    unsigned qb[NB][kSteps][2];
    float o[NB][kTiles][4];
    float m_run[NB][2], l_run[NB][2], factor[NB][2];  // of heads 2 j and 2 j + 1 of the eight
    float m_off[NB][2];                               // m_run - kLift, or 0 where nothing has been seen
    int left = ring.total;
    StageInfo u = {};
    for (int s = 0; left > 0; ++s) {
      const int slot = s % C::kStages;
      const unsigned known = ring.info[slot];
      const int keys = known & 0xff, last = known >> FourRing<C>::kLast & 3u;
      const unsigned blocks = known >> FourRing<C>::kBlocks & 0xffu;
      left -= (keys + kGrain - 1) / kGrain;
      if (known >> FourRing<C>::kFirst & 1u) {  // (while the copy is on its way)
        const int4 x = ring.units[slot];
        u.b = x.x, u.kvh = x.y, u.hb = x.z, u.uid = x.w;
        // Q as B fragments, fp16: a row is brought to a largest magnitude of 1 to 2 by a power of two, which leaves all of it
        // that counts: fp16 rows and bf16 ones lose nothing above 2^-14 of their largest element, and below it less than 2^-25 of that.
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          int b, h;
          const bool is = unit_row<RU>(a, u, nb * 8 + g, &b, &h);
          const T* const src = static_cast<const T*>(a.q) + (is ? static_cast<size_t>(b) * a.H + h : 0) * D;
          uint2 raw[kSteps];
#pragma unroll
          for (int st = 0; st < kSteps; ++st)
            raw[st] = is ? *reinterpret_cast<const uint2*>(src + Cols::k_column(st, j)) : make_uint2(0u, 0u);
          auto pair = [&](unsigned u) {
            if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&u));
            else return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
          };
          float most = 0.f;
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
            const float2 x = pair(raw[st].x), y = pair(raw[st].y);
            most = fmaxf(most, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
          }
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
          // 2^-e by the exponent's bits (rows of zeros, of what is below 2^-100 or not finite: as they are)
          const int e = static_cast<int>(__float_as_uint(most) >> 23) - 127;
          const bool plain = e < -100 || e > 127;
          const float down = plain ? 1.f : __uint_as_float(static_cast<unsigned>(127 - (e > 126 ? 126 : e)) << 23);
          const float up = plain ? 1.f : 1.f / down;
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
            const float2 x = pair(raw[st].x), y = pair(raw[st].y);
            qb[nb][st][0] = pack_pair<__half>(x.x * down, x.y * down);
            qb[nb][st][1] = pack_pair<__half>(y.x * down, y.y * down);
          }
          // (kept finite, so that scores of 0 stay 0 where queries and K's factor are beyond 32 bits together)
          const float f = fminf(up * (args.k_factor * a.scale_log2), 3.402823466e+38f);
          factor[nb][0] = __shfl_sync(0xffffffffu, f, 8 * j);
          factor[nb][1] = __shfl_sync(0xffffffffu, f, 8 * j + 4);
#pragma unroll
          for (int i = 0; i < kTiles; ++i) o[nb][i][0] = o[nb][i][1] = o[nb][i][2] = o[nb][i][3] = 0.f;
          m_run[nb][0] = m_run[nb][1] = -INFINITY;
          m_off[nb][0] = m_off[nb][1] = 0.f;
          l_run[nb][0] = l_run[nb][1] = 0.f;  // this lane's share of the sums
        }
      }
      if (!ring.wait(s)) return;
      const unsigned char *const k_tile = ring.tiles + 2 * slot * C::kTileBytes, *const v_tile = k_tile + C::kTileBytes;
#pragma unroll 1
      for (int key0 = 0; key0 < keys; key0 += 16 * kT) {
        constexpr unsigned kAll = (1u << kT) - 1u;
        const unsigned there = blocks >> (key0 / 16) & kAll;
        if (there == 0) continue;
        const bool whole = there == kAll && keys - key0 >= 16 * kT;  // (if not: see_of, keys of a tile that are there)
        auto see_of = [&](int t) { return (there >> t & 1u) ? keys - key0 - 16 * t : 0; };
        // S^T = K Q^T: keys g and g + 8 of a tile, heads 2 j and 2 j + 1
        float sc[kT][NB][4];
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) sc[t][nb][0] = sc[t][nb][1] = sc[t][nb][2] = sc[t][nb][3] = 0.f;
#pragma unroll
        for (int p = 0; p < kKPieces; ++p)
#pragma unroll
          for (int t = 0; t < kT; ++t) {
            const unsigned char* const k_codes = k_tile + (key0 + 16 * t) * C::kCodeBytes;
            const unsigned char* const k_scales = k_tile + C::SR * C::kCodeBytes + (key0 + 16 * t + key_g) * C::kScaleBytes;
            unsigned w[2][kKWords];
#pragma unroll
            for (int r = 0; r < 2; ++r) load_words(k_codes + k_at[p] + r * 8 * C::kCodeBytes, w[r]);
            // scales of the lane's blocks, two to a piece of 32 columns
            unsigned sk[2][2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const unsigned char* const at = k_scales + r * 8 * C::kScaleBytes;
              if constexpr (D >= 128) {
                const unsigned both = scales_to_half(static_cast<unsigned short>(load_u16(at + 2 * j + 8 * p)));
                sk[r][0] = __byte_perm(both, both, 0x1010);
                sk[r][1] = __byte_perm(both, both, 0x3232);
              } else {
                const unsigned one = at[D == 64 ? j : j / 2];
                sk[r][0] = sk[r][1] = scales_to_half(static_cast<unsigned short>(one | one << 8));
              }
            }
#pragma unroll
            for (int i = 0; i < kKWords; ++i) {
              unsigned h[2][4];
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                codes_to_half(w[r][i], h[r]);
#pragma unroll
                for (int e = 0; e < 4; ++e) h[r][e] = mul_half2(h[r][e], sk[r][i / 2]);
              }
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const unsigned ka[4] = {h[0][2 * e], h[1][2 * e], h[0][2 * e + 1], h[1][2 * e + 1]};
                const int st = p * 8 + 2 * i + e;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma16816<__half>(sc[t][nb], ka, qb[nb][st][0], qb[nb][st][1]);
              }
            }
          }
        // V's bytes are on their way while the weights are worked out, as far as the registers go
        constexpr bool kEarlyV = D * NB <= 128;
        unsigned vw[kT][2][2][kVWords], vs[kT][2][2];  // [tile][keys 2 j.., 2 j + 8..][key]: words of codes, bytes of scales
        auto load_v = [&](int t) {
          const unsigned char* const v_codes = v_tile + (key0 + 16 * t) * C::kCodeBytes;
          const unsigned char* const v_scales = v_tile + C::SR * C::kCodeBytes + (key0 + 16 * t) * C::kScaleBytes;
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const unsigned char* const at = v_codes + v_at[e] + r * 8 * C::kCodeBytes;
              if constexpr (D >= 64) load_words(at, vw[t][r][e]);
              else vw[t][r][e][0] = load_u16(at);
              const unsigned char* const of = v_scales + (e == 0 ? key_0 : key_1) * C::kScaleBytes + r * 8 * C::kScaleBytes;
              constexpr int kLanes = D == 256 ? 1 : 128 / D;  // lanes to a block
              if constexpr (D == 256) vs[t][r][e] = load_u16(of + 2 * g);
              else vs[t][r][e] = of[g / kLanes];
            }
        };
        if constexpr (kEarlyV) {
#pragma unroll
          for (int t = 0; t < kT; ++t) load_v(t);
        }
        bool more = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int t = 0; t < kT; ++t) {
            // (rounded before the difference to the reference, so that the largest score's is 0 however large it is)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[t][nb][i] *= factor[nb][i & 1];
            if (!whole) {
#pragma unroll
              for (int i = 0; i < 4; ++i) sc[t][nb][i] = key_g + (i < 2 ? 0 : 8) < see_of(t) ? sc[t][nb][i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) top[i & 1] = fmaxf(top[i & 1], sc[t][nb][i]);
          }
          // (the difference is exact where the sum may round to a score a step of 2^4 above the reference: a weight of 2^16)
          more = more || top[0] - m_run[nb][0] > kSlack || top[1] - m_run[nb][1] > kSlack;
        }
        if (__any_sync(0xffffffffu, more)) {  // rare after a unit's first keys
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float f[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = -INFINITY;
#pragma unroll
              for (int t = 0; t < kT; ++t) mx = fmaxf(mx, fmaxf(sc[t][nb][c], sc[t][nb][2 + c]));
#pragma unroll
              for (int d = 4; d < 32; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
              const float mn = fmaxf(m_run[nb][c], mx);
              const float off = mn == -INFINITY ? 0.f : mn - kLift;
              f[c] = m_run[nb][c] == -INFINITY ? 0.f : ex2(m_off[nb][c] - off);
              l_run[nb][c] = m_run[nb][c] == -INFINITY ? l_run[nb][c] : l_run[nb][c] * f[c];  // (0, or NaN to keep)
              m_run[nb][c] = mn;
              m_off[nb][c] = off;
            }
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
              o[nb][i][0] *= f[0];
              o[nb][i][1] *= f[1];
              o[nb][i][2] *= f[0];
              o[nb][i][3] *= f[1];
            }
          }
        }
        // P^T as the B fragments of the second product, rounded to fp16 (l is not): off by 2^-11 of a weight, or by 2^-32 of the reference's
        unsigned pb[kT][NB][2];
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = ex2(sc[t][nb][i] - m_off[nb][i & 1]);
            l_run[nb][0] += p[0] + p[2];
            l_run[nb][1] += p[1] + p[3];
            pb[t][nb][0] = transposed(pack_pair<__half>(p[0], p[1]));
            pb[t][nb][1] = transposed(pack_pair<__half>(p[2], p[3]));
          }
        // O^T += V^T P^T
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          if constexpr (!kEarlyV) load_v(t);
          unsigned h[2][kVWords][2][4], sv[2][2];  // [keys 2 j.., 2 j + 8..]: the codes of two keys, column by column; the scales
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            auto& w = vw[t][r];
            // the scales of the two keys, of the block of row g and of that of row g + 8 (head_dim 256: the next block); 0 for
            // keys that are not the sequence's, whose bytes may be anything
            unsigned s0 = vs[t][r][0], s1 = vs[t][r][1];
            if (!whole) {
              s0 = key_0 + 8 * r < see_of(t) ? s0 : 0u;
              s1 = key_1 + 8 * r < see_of(t) ? s1 : 0u;
            }
            if constexpr (D == 256) {
              const unsigned both = __byte_perm(s0, s1, 0x5140);  // (s0.lo, s1.lo, s0.hi, s1.hi)
              sv[r][0] = scales_to_half(static_cast<unsigned short>(both));
              sv[r][1] = scales_to_half(static_cast<unsigned short>(both >> 16));
            } else {
              sv[r][0] = sv[r][1] = scales_to_half(static_cast<unsigned short>(__byte_perm(s0, s1, 0x0040)));
            }
            // the codes of the two keys change places so that those of a column lie in a byte
#pragma unroll
            for (int i = 0; i < kVWords; ++i) {
              const unsigned even = (w[0][i] & 0x0f0f0f0fu) | ((w[1][i] << 4) & 0xf0f0f0f0u);
              const unsigned odd = ((w[0][i] >> 4) & 0x0f0f0f0fu) | (w[1][i] & 0xf0f0f0f0u);
              codes_to_half(even, h[r][i][0]);
              codes_to_half(odd, h[r][i][1]);
            }
          }
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            constexpr int x = Cols::v_other;  // from the column of row g to that of row g + 8
            const unsigned av[4] = {mul_half2(h[0][i / 8][i % 2][i % 8 / 2], sv[0][0]), mul_half2(h[0][(i + x) / 8][(i + x) % 2][(i + x) % 8 / 2], sv[0][1]),
                                    mul_half2(h[1][i / 8][i % 2][i % 8 / 2], sv[1][0]), mul_half2(h[1][(i + x) / 8][(i + x) % 2][(i + x) % 8 / 2], sv[1][1])};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma16816<__half>(o[nb][i], av, pb[t][nb][0], pb[t][nb][1]);
          }
        }
      }
      __syncwarp();
      ring.copy(slot);
      if (last) {
        const size_t part = (static_cast<size_t>(blockIdx.x) * C::kWarps + warp + u.uid) * a.rs;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float l = l_run[nb][c];
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
            const int r = nb * 8 + 2 * j + c;
            int b, h;
            if (!unit_row<RU>(a, u, r, &b, &h)) continue;
            const bool result = last == 2;
            const float f = !result ? args.v_factor : l == 0.f ? 0.f : args.v_factor / l;  // (no key seen: O is 0 as well)
            constexpr int kEach = D / 16;  // columns side by side of row g, as many of row g + 8 behind them
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int col = Cols::v_column(0, g) + x * Cols::v_other;
              if (result) {
                T* const dst = static_cast<T*>(a.out) + (static_cast<size_t>(b) * a.H + h) * D + col;
#pragma unroll
                for (int i = 0; i < kEach; i += 2)
                  *reinterpret_cast<unsigned*>(dst + i) = pack_pair<T>(o[nb][i][2 * x + c] * f, o[nb][i + 1][2 * x + c] * f);
              } else {
                float* const dst = a.part_o + (part + r) * D + col;
#pragma unroll
                for (int i = 0; i < kEach; i += 2)
                  *reinterpret_cast<float2*>(dst + i) = make_float2(o[nb][i][2 * x + c] * f, o[nb][i + 1][2 * x + c] * f);
              }
            }
            if (g == 0) {
              if (!result) a.part_ml[part + r] = make_float2(m_run[nb][c] == -INFINITY ? -INFINITY : m_off[nb][c], l);
              else if (a.lse)
                a.lse[static_cast<size_t>(b) * a.H + h] = l > 0.f ? m_off[nb][c] * kLn2 + logf(l) : l == 0.f ? -INFINITY : l;
            }
          }
      }
    }
  };
  // (behind a launch that gave up nothing is computed; the fold writes nothing then either)
  if (ring.total > 0 && a.missing >= 0 && __shfl_sync(0xffffffffu, *reinterpret_cast<volatile int*>(a.status), 0) == 0) walk();
  __syncthreads();
  if (*gave_up) {  // give copies in flight time to land
    const unsigned long long t0 = tcgen::global_ns();
    while (tcgen::global_ns() - t0 < 1000000ull) __nanosleep(1000);
  }
}

// ---- rows back out of a cache --------------------------------------------------------

struct ReadRows {
  char* data;
  long long row, head;  // strides in elements
};
struct ReadArgs {
  const char* pages[2];  // k, v
  ReadRows out[2];
  const int* table;
  long long table_stride;
  const int* ends;   // sequence b's rows are rows ends[b] to ends[b + 1] of the results
  const int* start;  // the first of them in the cache (NULL: 0)
  int rows, num_pages, max_pages, shift, B, kvH;
  int vec;           // every row of the results is 16-byte aligned
  float factor[2];
};

// A block has as many rows of the results as threads share out: it finds out whose they are and where, and a thread copies 16 bytes of a
// row, or (4 bits) one block of 16 elements, for one head after the other, `per` of the list of K's heads and V's, four at a time. Bound
// by memory, a row comes in once and goes out once: 541 MB out of 4 bits 92 us, 0.90 of the copy's rate.
constexpr int kReadThreads = 256, kReadAhead = 4;
template <typename T, bool kFour>
constexpr int read_pieces(int D) { return kFour ? D / 16 : D * static_cast<int>(sizeof(T)) / 16; }

template <typename T, int D, bool kFour>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(const __grid_constant__ ReadArgs a, int per) {
  constexpr int kPieces = read_pieces<T, kFour>(D), kTokens = kReadThreads / kPieces, kEach = D / kPieces;
  constexpr int kWords = kEach * static_cast<int>(sizeof(T)) / 4;
  __shared__ long long place_of[kTokens];
  let_next_start();
  wait_for_previous();
  const int token0 = static_cast<int>(blockIdx.x) * kTokens;
  if (threadIdx.x < kTokens) {
    const int i = token0 + static_cast<int>(threadIdx.x);
    long long place = -2;  // a row of the results that is no sequence's stays as it is
    if (i < a.rows && i >= a.ends[0] && i < a.ends[a.B]) {
      int lo = 0, hi = a.B;  // ends[lo] <= i < ends[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.ends[mid] <= i) lo = mid;
        else hi = mid;
      }
      place = paged_row(a.table + lo * a.table_stride, a.max_pages, a.num_pages, a.shift, a.kvH,
                        static_cast<long long>(a.start ? a.start[lo] : 0) + (i - a.ends[lo]));
    }
    place_of[threadIdx.x] = place;
  }
  __syncthreads();
  const int token = threadIdx.x / kPieces, piece = threadIdx.x % kPieces;
  const long long place = place_of[token];
  if (place == -2) return;
  const bool there = place >= 0;  // (a row that there is not is zeros)
  const int row = static_cast<int>(place) & ((1 << a.shift) - 1);
  const size_t page_head = there ? static_cast<size_t>(place >> a.shift) : 0;
  [[maybe_unused]] const int code_at = row * (D / 2) + ((piece / 2) ^ four_turn(row, D)) * 16 + piece % 2 * 8;
  [[maybe_unused]] const int scale_at = (D / 2 << a.shift) + row * (D / 16) + piece;
  const int end = min((static_cast<int>(blockIdx.y) + 1) * per, 2 * a.kvH);
  for (int h0 = static_cast<int>(blockIdx.y) * per; h0 < end; h0 += kReadAhead) {
    unsigned u[kReadAhead][kFour ? 3 : 4];
#pragma unroll
    for (int n = 0; n < kReadAhead; ++n) {
#pragma unroll
      for (int w = 0; w < (kFour ? 3 : 4); ++w) u[n][w] = 0u;
      if (h0 + n >= end || !there) continue;
      const bool v = h0 + n >= a.kvH;
      const size_t head = page_head + (h0 + n - (v ? a.kvH : 0));
      const char* const pages = v ? a.pages[1] : a.pages[0];
      if constexpr (kFour) {
        const char* const from = pages + (head << a.shift) * four_row_bytes(D);
        const uint2 c = *reinterpret_cast<const uint2*>(from + code_at);
        u[n][0] = c.x, u[n][1] = c.y;
        u[n][2] = static_cast<unsigned char>(from[scale_at]);
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(pages + (((head << a.shift) + row) * D + piece * kEach) * sizeof(T));
        u[n][0] = x.x, u[n][1] = x.y, u[n][2] = x.z, u[n][3] = x.w;
      }
    }
#pragma unroll
    for (int n = 0; n < kReadAhead; ++n) {
      if (h0 + n >= end) break;
      const bool v = h0 + n >= a.kvH;
      const ReadRows& out = v ? a.out[1] : a.out[0];
      T* const dst = reinterpret_cast<T*>(out.data) + static_cast<long long>(token0 + token) * out.row +
                     (h0 + n - (v ? a.kvH : 0)) * out.head + piece * kEach;
      unsigned w[kWords];
      if constexpr (kFour) {
        const unsigned s = scales_to_half(static_cast<unsigned short>(u[n][2] | u[n][2] << 8));
        const float f = v ? a.factor[1] : a.factor[0];
        unsigned h[2][4];
        codes_to_half(u[n][0], h[0]);
        codes_to_half(u[n][1], h[1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned x = mul_half2(h[e / 4][e % 4], s);
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&x));
          w[e] = pack_pair<T>(y.x * f, y.y * f);
        }
      } else {
#pragma unroll
        for (int e = 0; e < kWords; ++e) w[e] = u[n][e];
      }
      if constexpr (kFour) {
        // Two lanes have 64 bytes side by side; they exchange halves, so that a store of the warp has whole 32-byte sectors (four prompts of
        // 20000 to 32768 rows, 8 KV heads of 128 in bf16: 127 -> 92 us).
        if (a.vec) {
          const bool odd = threadIdx.x & 1;
          unsigned r[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = __shfl_xor_sync(0xffffffffu, odd ? w[e] : w[4 + e], 1);
          uint4* const to = reinterpret_cast<uint4*>(dst) - (odd ? 2 : 0) + (odd ? 1 : 0);  // (of the even lane's block, and 32 bytes behind it)
          to[0] = odd ? make_uint4(r[0], r[1], r[2], r[3]) : make_uint4(w[0], w[1], w[2], w[3]);
          to[2] = odd ? make_uint4(w[4], w[5], w[6], w[7]) : make_uint4(r[0], r[1], r[2], r[3]);
          continue;
        }
      }
      if (a.vec) {
#pragma unroll
        for (int e = 0; e < kWords; e += 4) reinterpret_cast<uint4*>(dst)[e / 4] = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
      } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < kWords; ++e) dst[e] = __uint_as_float(w[e]);
      } else {
        unsigned short* const to = reinterpret_cast<unsigned short*>(dst);
#pragma unroll
        for (int e = 0; e < kWords; ++e) to[2 * e] = static_cast<unsigned short>(w[e]), to[2 * e + 1] = static_cast<unsigned short>(w[e] >> 16);
      }
    }
  }
}

// ---- host side ----------------------------------------------------------------------

struct FourPlan {
  int NB, HB, blocks, warps, rs;
  double most;  // stages that there can be
  size_t unit_bytes, ml_bytes, bytes;
};

FourPlan make_plan(const ra_paged_kv& c, int heads) {
  FourPlan p = {};
  const int G = (heads + c.kv_heads - 1) / c.kv_heads;
  p.NB = G > 8 ? 2 : 1;
  p.HB = (G + 8 * p.NB - 1) / (8 * p.NB);
  p.warps = four_warps(c.head_dim, p.NB);
  const size_t units = static_cast<size_t>(c.kv_heads) * c.batch * p.HB;
  const long long room = static_cast<long long>(c.max_pages) * c.page_size;
  p.most = static_cast<double>(units) * ((room + kGrain - 1) / kGrain);
  const int wave = kBlocksPerSm * sm_count();
  p.blocks = p.most < static_cast<double>(wave) * p.warps ? (static_cast<int>(p.most) + p.warps - 1) / p.warps : wave;
  p.rs = std::min(8 * p.NB, G);
  auto whole = [](size_t n) { return (n + 127) & ~static_cast<size_t>(127); };
  const size_t rows = (units + static_cast<size_t>(p.blocks) * p.warps) * p.rs;
  p.unit_bytes = whole(units * sizeof(int2));
  p.ml_bytes = whole(rows * sizeof(float2));
  p.bytes = p.unit_bytes + p.ml_bytes + rows * c.head_dim * sizeof(float);
  return p;
}

template <typename T, int D, int NB>
int launch_four(const FourArgs& a, const FourPlan& p, cudaStream_t stream) {
  if (p.blocks > 0) {
    const int rc = launch_main<paged_4bit_kernel<T, D, NB>, FourBlock<D, NB>>(p.blocks, stream, a);
    if (rc != RA_OK) return rc;
  }
  return launch_fold<T, D, 8 * NB>(a.p, stream);
}

bool power_of_two(float f) { return f >= 1.0f / (1 << 30) && f <= 1 << 30 && std::exp2(std::round(std::log2(f))) == f; }

}  // namespace

int check_paged_4bit(const ra_paged_kv& c, float k_scale, float v_scale, const char* what) {
  RAB_REQUIRE(c.dtype == RA_F16 || c.dtype == RA_BF16, RA_ERR_INVALID, "%s: rows are fp16 or bf16, got dtype %d", what, c.dtype);
  RAB_REQUIRE(c.head_dim == 32 || c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, RA_ERR_UNSUPPORTED,
              "%s: unsupported head_dim=%d (supported: 32, 64, 128, 256)", what, c.head_dim);
  RAB_REQUIRE(power_of_two(k_scale) && power_of_two(v_scale), RA_ERR_INVALID,
              "%s: k_scale and v_scale are powers of two from 2^-30 to 2^30", what);
  return check_paged(c, what);
}

namespace {

int check_decode(const ra_paged_kv& c, int heads, float k_scale, float v_scale) {
  const char* const what = "paged_decode_4bit";
  const int rc = check_paged_4bit(c, k_scale, v_scale, what);
  if (rc != RA_OK) return rc;
  RAB_REQUIRE(heads >= c.kv_heads && heads <= 4096, RA_ERR_INVALID, "%s: bad heads", what);
  RAB_REQUIRE(static_cast<long long>(c.batch) * heads < (1ll << 24), RA_ERR_INVALID, "%s: too many rows", what);
  RAB_REQUIRE(static_cast<long long>(c.num_pages) * c.kv_heads < (1ll << 31) - 1, RA_ERR_INVALID, "%s: too many pages", what);
  return RA_OK;
}

// The entry points that read rows back. `kFour`: out of a cache in 4 bits.
template <bool kFour>
int read_rows(const char* what, const ra_paged_kv* cache, float k_scale, float v_scale, const int* ends, const int* start,
              const ra_rows* k_out, const ra_rows* v_out, int rows, cudaStream_t stream) {
  RAB_REQUIRE(cache && k_out && v_out, RA_ERR_INVALID, "%s: null argument", what);
  ra_paged_kv c = *cache;
  c.lens = ends;  // (lengths are not read)
  int rc = RA_OK;
  if (kFour) {
    rc = check_paged_4bit(c, k_scale, v_scale, what);
  } else {
    RAB_REQUIRE(c.dtype == RA_F32 || c.dtype == RA_F16 || c.dtype == RA_BF16, RA_ERR_INVALID, "%s: unknown dtype %d", what, c.dtype);
    RAB_REQUIRE(c.head_dim == 32 || c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, RA_ERR_UNSUPPORTED,
                "%s: unsupported head_dim=%d (supported: 32, 64, 128, 256)", what, c.head_dim);
    rc = check_paged(c, what);
  }
  if (rc == RA_OK) rc = check_lists(c, what);
  if (rc != RA_OK) return rc;
  RAB_REQUIRE(rows >= 0, RA_ERR_INVALID, "%s: bad shape", what);
  RAB_REQUIRE(c.kv_heads <= 1 << 16, RA_ERR_INVALID, "%s: bad heads", what);
  if (c.batch == 0 || rows == 0) return RA_OK;
  const int es = c.dtype == RA_F32 ? 4 : 2;
  RAB_REQUIRE(k_out->data && v_out->data, RA_ERR_INVALID, "%s: null argument", what);
  RAB_REQUIRE(((reinterpret_cast<uintptr_t>(k_out->data) | reinterpret_cast<uintptr_t>(v_out->data)) & (es - 1u)) == 0 &&
                  (reinterpret_cast<uintptr_t>(start) & 3u) == 0,
              RA_ERR_INVALID, "%s: rows or start are not aligned to their elements", what);
  RAB_REQUIRE(rows_apart(*k_out, c.head_dim, c.kv_heads, rows) && rows_apart(*v_out, c.head_dim, c.kv_heads, rows), RA_ERR_INVALID,
              "%s: rows of a result overlap", what);
  ReadArgs a;
  std::memset(&a, 0, sizeof(a));
  const ra_rows* out[2] = {k_out, v_out};
  unsigned long long all = 0;
  for (int i = 0; i < 2; ++i) {
    a.out[i] = {static_cast<char*>(out[i]->data), out[i]->row_stride, out[i]->head_stride};
    all |= reinterpret_cast<uintptr_t>(out[i]->data);
    if (rows > 1) all |= static_cast<unsigned long long>(out[i]->row_stride) * es;
    if (c.kv_heads > 1) all |= static_cast<unsigned long long>(out[i]->head_stride) * es;
  }
  a.vec = (all & 15u) == 0;
  a.pages[0] = static_cast<const char*>(c.k);
  a.pages[1] = static_cast<const char*>(c.v);
  a.table = c.page_table;
  a.table_stride = c.table_stride;
  a.ends = ends;
  a.start = start;
  a.rows = rows;
  a.num_pages = c.num_pages;
  a.max_pages = c.max_pages;
  a.shift = page_shift(c.page_size);
  a.B = c.batch;
  a.kvH = c.kv_heads;
  a.factor[0] = k_scale;
  a.factor[1] = v_scale;
  auto go = [&](auto t, auto d) -> int {
    constexpr unsigned kTokens = kReadThreads / read_pieces<decltype(t), kFour>(d());
    const unsigned blocks = (static_cast<unsigned>(rows) + kTokens - 1) / kTokens;
    // all heads a block, whose place it finds but once, or, where that leaves SMs without enough blocks, fewer
    const int heads = 2 * c.kv_heads, room = 8 * sm_count();
    int per = heads;
    while (per > kReadAhead && static_cast<long long>(blocks) * ((heads + per - 1) / per) < room) per = (per + 1) / 2;
    RAB_REQUIRE((heads + per - 1) / per <= 65535, RA_ERR_INVALID, "%s: bad heads", what);
    RAB_CUDA(launch_overlapped(paged_read_kernel<decltype(t), d(), kFour>, dim3(blocks, static_cast<unsigned>((heads + per - 1) / per)),
                               dim3(kReadThreads), 0, stream, a, per));
    return RA_OK;
  };
  auto by_dim = [&](auto t) -> int {
    if (c.head_dim == 32) return go(t, std::integral_constant<int, 32>());
    if (c.head_dim == 64) return go(t, std::integral_constant<int, 64>());
    if (c.head_dim == 128) return go(t, std::integral_constant<int, 128>());
    return go(t, std::integral_constant<int, 256>());
  };
  if constexpr (!kFour) {
    if (c.dtype == RA_F32) return by_dim(float());
  }
  return c.dtype == RA_BF16 ? by_dim(__nv_bfloat16()) : by_dim(__half());
}

}  // namespace
}  // namespace rab

using namespace rab;

extern "C" {

size_t ra_paged_decode_4bit_workspace_bytes(const ra_paged_kv* cache, int heads) {
  if (!cache || check_decode(*cache, heads, 1.f, 1.f) != RA_OK) return 0;
  ra_paged_kv c = *cache;
  if (c.num_pages == 0) c.max_pages = 0;
  return make_plan(c, heads).bytes;
}

int ra_paged_decode_4bit(const ra_paged_kv* cache, float k_scale, float v_scale, const void* q, int heads, void* out, float* lse,
                         void* workspace, size_t workspace_bytes, ra_stream stream_) {
  const char* const what = "paged_decode_4bit";
  RAB_REQUIRE(cache != nullptr, RA_ERR_INVALID, "%s: null argument", what);
  int rc = check_decode(*cache, heads, k_scale, v_scale);
  if (rc == RA_OK) rc = check_lists(*cache, what);
  if (rc != RA_OK) return rc;
  if (cache->batch == 0) return RA_OK;
  RAB_REQUIRE(q && out, RA_ERR_INVALID, "%s: null argument", what);
  RAB_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0, RA_ERR_INVALID,
              "%s: q and out must be 16-byte aligned", what);
  RAB_REQUIRE((reinterpret_cast<uintptr_t>(lse) & 3u) == 0, RA_ERR_INVALID, "%s: lse is not aligned to its elements", what);
  ra_paged_kv c = *cache;
  if (c.num_pages == 0) c.max_pages = 0;  // (holds no keys, whatever the tables say)
  const FourPlan p = make_plan(c, heads);
  RAB_REQUIRE(p.most < 2147483648.0 * std::max(p.blocks * p.warps, 1), RA_ERR_INVALID, "%s: too many keys", what);
  RAB_REQUIRE(workspace && workspace_bytes >= p.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, RA_ERR_OVERFLOW,
              "%s: workspace too small or not 16-byte aligned", what);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  unsigned char* const ws = static_cast<unsigned char*>(workspace);
  FourArgs f;
  std::memset(&f, 0, sizeof(f));
  f.k_factor = k_scale;
  f.v_factor = v_scale;
  PagedArgs& a = f.p;
  a.q = q;
  a.k = c.k;
  a.v = c.v;
  a.out = out;
  a.lse = lse;
  a.table = c.page_table;
  a.table_stride = c.table_stride;
  a.lens = c.lens;
  a.num_pages = c.num_pages;
  a.max_pages = c.max_pages;
  a.shift = page_shift(c.page_size);
  a.B = c.batch;
  a.H = heads;
  a.kvH = c.kv_heads;
  a.G = (heads + c.kv_heads - 1) / c.kv_heads;
  a.HB = p.HB;
  a.rs = p.rs;
  a.scale_log2 = kLog2e / std::sqrt(static_cast<float>(c.head_dim));
  a.unit_parts = reinterpret_cast<int2*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + p.unit_bytes);
  a.part_o = reinterpret_cast<float*>(ws + p.unit_bytes + p.ml_bytes);
  a.status = device_status_ptr();
  RAB_REQUIRE(a.status != nullptr, RA_ERR_CUDA, "%s: no device status word", what);
  a.wait_ns = tcgen::tc_wait_limit_ns();
  a.shares = p.blocks * p.warps;
  const int stall = tcgen::tc_stall_after();
  a.missing = stall > 0 ? 16 : stall == 0 ? -1 : 0;
  auto go = [&](auto t, auto d) -> int {
    using T = decltype(t);
    return p.NB == 1 ? launch_four<T, d(), 1>(f, p, stream) : launch_four<T, d(), 2>(f, p, stream);
  };
  auto by_dim = [&](auto t) -> int {
    if (c.head_dim == 32) return go(t, std::integral_constant<int, 32>());
    if (c.head_dim == 64) return go(t, std::integral_constant<int, 64>());
    if (c.head_dim == 128) return go(t, std::integral_constant<int, 128>());
    return go(t, std::integral_constant<int, 256>());
  };
  return c.dtype == RA_BF16 ? by_dim(__nv_bfloat16()) : by_dim(__half());
}

int ra_paged_read(const ra_paged_kv* cache, const int* ends, const int* start, const ra_rows* k_out, const ra_rows* v_out, int rows,
                  ra_stream stream) {
  return read_rows<false>("paged_read", cache, 1.f, 1.f, ends, start, k_out, v_out, rows, static_cast<cudaStream_t>(stream));
}

int ra_paged_read_4bit(const ra_paged_kv* cache, float k_scale, float v_scale, const int* ends, const int* start,
                       const ra_rows* k_out, const ra_rows* v_out, int rows, ra_stream stream) {
  return read_rows<true>("paged_read_4bit", cache, k_scale, v_scale, ends, start, k_out, v_out, rows, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
