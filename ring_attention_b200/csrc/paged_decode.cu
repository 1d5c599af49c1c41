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
#include "paged_walk.cuh"

namespace rab {

namespace {

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

// ---- host side ----------------------------------------------------------------------

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
