// Rows of queries and keys on their way into attention: the norm of each head's row, the position rotation, and, for a paged
// cache, the place a row goes to; and the backward pass of norm and rotation.
//
//   y = R_p (x r w),  r = (mean(x^2) + eps)^-1/2,  R_p turns pair i by p f_i
//   backward, with g = R_-p dy:  dw = sum over rows of g x r,  dx = r (g w - x r^2 mean(g w x))
//
// All of it is bound by memory: a row comes in once and goes out once. A lane holds 16 bytes of a row (32 of an fp32 row of
// 256), so 4 to 32 lanes share a row and a warp takes several heads of one token at a time. cos and sin of the token's position
// are worked out once for all heads that the warp takes, from an angle in fixed point (see ra_rope), and multiplied by the
// weights ahead of the rows: a row then costs a sum of squares and two multiply-adds an element. With pairs half a row apart the
// partner's elements come by shuffles of the raw words, with neighbouring pairs they are the lane's own.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace rab {

namespace {

constexpr int kWarps = 8;

// E elements of a row to a lane, L lanes to a row, R rows to a warp.
template <typename T, int D>
struct RowCfg {
  static constexpr int E = D * static_cast<int>(sizeof(T)) > 512 ? D / 32 : 16 / static_cast<int>(sizeof(T));
  static constexpr int L = D / E;
  static constexpr int R = 32 / L;
  static constexpr int kWords = E * static_cast<int>(sizeof(T)) / 4;  // 32-bit words of a lane
};

template <typename T>
__device__ inline float2 unpack2(unsigned u);
template <>
__device__ inline float2 unpack2<__half>(unsigned u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ inline float2 unpack2<__nv_bfloat16>(unsigned u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <typename T, int E>
__device__ inline void unpack(const unsigned* u, float (&x)[E]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 f = unpack2<T>(u[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ inline unsigned pack2(float a, float b);
template <>
__device__ inline unsigned pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <>
__device__ inline unsigned pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <typename T, int E>
__device__ inline void pack(const float (&x)[E], unsigned* u) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < E; ++i) u[i] = __float_as_uint(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) u[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
  }
}

// A lane's words of a row: 16 bytes at a time, or (`vec` false: some row is not 16-byte aligned) an element at a time.
template <typename T, int W>
__device__ inline void load_words(const T* p, bool vec, unsigned (&u)[W]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned*>(p) + 4 * i);
      u[4 * i] = v.x, u[4 * i + 1] = v.y, u[4 * i + 2] = v.z, u[4 * i + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < W; ++i) u[i] = __float_as_uint(p[i]);
  } else {
    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) u[i] = s[2 * i] | static_cast<unsigned>(s[2 * i + 1]) << 16;
  }
}
template <typename T, int W>
__device__ inline void store_words(T* p, bool vec, const unsigned (&u)[W]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i)
      *reinterpret_cast<uint4*>(reinterpret_cast<unsigned*>(p) + 4 * i) =
          make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < W; ++i) p[i] = __uint_as_float(u[i]);
  } else {
    unsigned short* s = reinterpret_cast<unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      s[2 * i] = static_cast<unsigned short>(u[i]);
      s[2 * i + 1] = static_cast<unsigned short>(u[i] >> 16);
    }
  }
}

struct Rows {
  char* data;
  long long batch, head, row;  // strides in elements
  int vec;                     // every row is 16-byte aligned
};

struct Args {
  Rows in[3], dy[2], out[3];  // q, k, v (v and a cache's k_out, v_out: see paged below)
  int heads[3];               // 0: that side is absent
  int B, S;
  const void* w[2];
  int w_f32;
  float eps;
  int rot_dim;  // 0: no rotation
  PosMap map;
  int pos_stride;
  const int* positions;
  long long pos_batch;
  // paged: rows go to lens[b] + t
  const int* lens;
  const int* counts;
  const int* table;
  long long table_stride;
  int num_pages, max_pages, page_shift;
  float* part;  // backward: partial sums of the weights' gradients, [block][2][D]
  unsigned long long turns[RA_ROPE_MAX_PAIRS];
};

__device__ inline float weight_at(const void* w, int w_f32, int i, float) { return static_cast<const float*>(w)[i]; }
__device__ inline float weight_at(const void* w, int w_f32, int i, __half) {
  return w_f32 ? static_cast<const float*>(w)[i] : __half2float(static_cast<const __half*>(w)[i]);
}
__device__ inline float weight_at(const void* w, int w_f32, int i, __nv_bfloat16) {
  return w_f32 ? static_cast<const float*>(w)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

__device__ inline long long row_position(const Args& a, int b, int s) {
  if (a.positions) return a.positions[b * a.pos_batch + s];
  if (a.lens) return static_cast<long long>(a.lens[b]) + s;
  const int seg = s / a.map.seg_len;
  return a.map.base[seg] + static_cast<long long>(s - seg * a.map.seg_len) * a.pos_stride;
}

// The place of a lane's elements in the rotation: its partner's lane, and (cos, signed sin) of its elements, so that
// y[e] = x[e] c[e] + partner[e] s[e].
template <typename T, int D, bool kInter>
struct Turn {
  using C = RowCfg<T, D>;
  static constexpr int E = C::E;
  int partner;  // lane; its own where nothing turns
  bool turns;
  float c[E], s[E];
  __device__ inline void place(const Args& a, int lane) {
    const int at = lane % C::L * E, half = a.rot_dim / 2;
    turns = at < a.rot_dim;
    partner = kInter || !turns ? lane : at < half ? lane + half / E : lane - half / E;
  }
  __device__ inline void angles(const Args& a, int lane, long long pos) {
    const int at = lane % C::L * E, half = a.rot_dim / 2;
#pragma unroll
    for (int e = 0; e < E; ++e) c[e] = 1.f, s[e] = 0.f;
    if (!turns) return;
    // (the angle in half turns, from the upper word of its place in the turn: off by 2^-25 of a half turn at most)
    auto angle = [&](int pair, float* si, float* co) {
      const unsigned long long t = static_cast<unsigned long long>(pos) * a.turns[pair];
      sincospif(static_cast<float>(static_cast<int>(t >> 32)) * 4.656612873077393e-10f, si, co);
    };
    if constexpr (kInter) {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float si, co;
        angle((at + e) / 2, &si, &co);
        c[e] = c[e + 1] = co;
        s[e] = -si;
        s[e + 1] = si;
      }
    } else {
      const int first = at < half ? at : at - half;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float si, co;
        angle(first + e, &si, &co);
        c[e] = co;
        s[e] = at < half ? -si : si;
      }
    }
  }
  // The partner's elements of a row whose words are u and whose elements are x (every lane of the warp calls).
  __device__ inline void other(const unsigned (&u)[C::kWords], const float (&x)[E], float (&xp)[E]) const {
    if constexpr (kInter) {
#pragma unroll
      for (int e = 0; e < E; ++e) xp[e] = x[e ^ 1];
    } else {
      unsigned up[C::kWords];
#pragma unroll
      for (int i = 0; i < C::kWords; ++i) up[i] = __shfl_sync(0xffffffffu, u[i], partner);
      unpack<T, E>(up, xp);
    }
  }
};

template <int L>
__device__ inline float row_sum(float v) {
#pragma unroll
  for (int i = L / 2; i > 0; i /= 2) v += __shfl_xor_sync(0xffffffffu, v, i);
  return v;
}

// A warp takes `per` groups of R rows of one token, from the list of q's groups, then k's, then v's.
template <typename T, int D, bool kInter, bool kPaged>
__global__ void __launch_bounds__(kWarps * 32) norm_rope_kernel(const __grid_constant__ Args a, long long total, int per) {
  using C = RowCfg<T, D>;
  constexpr int E = C::E, W = C::kWords, kAhead = 4;
  const int lane = threadIdx.x & 31, sub = lane / C::L, at = lane % C::L * E;
  const long long id = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  let_next_start();
  wait_for_previous();
  if (id >= total) return;
  const long long tokens = static_cast<long long>(a.B) * a.S;
  const int chunk = static_cast<int>(id / tokens);
  const long long token = id - chunk * tokens;
  const int b = static_cast<int>(token / a.S), t = static_cast<int>(token - static_cast<long long>(b) * a.S);
  long long place = -1;  // paged: row of the cache's first head that takes the token's K and V
  if constexpr (kPaged) {
    if (a.counts && t >= a.counts[b]) return;
    place = paged_row(a.table + b * a.table_stride, a.max_pages, a.num_pages, a.page_shift, a.heads[1],
                      static_cast<long long>(a.lens[b]) + t);
  }
  Turn<T, D, kInter> turn;
  turn.place(a, lane);
  turn.angles(a, lane, a.rot_dim ? row_position(a, b, t) : 0);
  const int beg = chunk * per, end = beg + per;
  int first = 0;  // group of a side's first row
#pragma unroll
  for (int side = 0; side < (kPaged ? 3 : 2); ++side) {
    const int heads = a.heads[side], groups = (heads + C::R - 1) / C::R;
    const int lo = max(beg - first, 0), hi = min(end - first, groups);
    first += groups;
    if (lo >= hi) continue;
    const Rows in = a.in[side], out = a.out[side];
    const bool to_cache = kPaged && side > 0;
    if (to_cache && place < 0) continue;
    const T* src = reinterpret_cast<const T*>(in.data) + b * in.batch + t * in.row + at;
    T* dst = reinterpret_cast<T*>(out.data) + (to_cache ? place * D : b * out.batch + t * out.row) + at;
    const long long out_head = to_cache ? static_cast<long long>(D) << a.page_shift : out.head;
    const bool norm = side < 2 && a.w[side < 2 ? side : 0] != nullptr;
    // factors of the element and of its partner, weights included
    float fx[E], fp[E];
    if (side < 2) {
      const int p_at = kInter ? at : turn.partner % C::L * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        fx[e] = turn.c[e] * (norm ? weight_at(a.w[side], a.w_f32, at + e, T()) : 1.f);
        fp[e] = turn.s[e] * (norm ? weight_at(a.w[side], a.w_f32, p_at + (kInter ? e ^ 1 : e), T()) : 1.f);
      }
    }
    for (int g = lo; g < hi; g += kAhead) {
      unsigned u[kAhead][W];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int h = (g + i) * C::R + sub;
#pragma unroll
        for (int j = 0; j < W; ++j) u[i][j] = 0;
        if (g + i < hi && h < heads) load_words<T, W>(src + h * in.head, in.vec, u[i]);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (g + i >= hi) break;
        const int h = (g + i) * C::R + sub;
        if (side < 2) {
          float x[E], xp[E], y[E];
          unpack<T, E>(u[i], x);
          float r = 1.f;
          if (norm) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) sum = fmaf(x[e], x[e], sum);
            r = rsqrtf(row_sum<C::L>(sum) * (1.f / D) + a.eps);
          }
          turn.other(u[i], x, xp);
#pragma unroll
          for (int e = 0; e < E; ++e) y[e] = r * (turn.turns ? fmaf(x[e], fx[e], xp[e] * fp[e]) : x[e] * fx[e]);
          pack<T, E>(y, u[i]);
        }
        if (h < heads) store_words<T, W>(dst + h * out_head, out.vec, u[i]);
      }
    }
  }
}

// The backward pass: a warp walks over tokens, all heads of each, and keeps its share of the weights' gradients; the block's
// sums go to its place in the workspace, in an order that does not depend on timing.
template <typename T, int D, bool kInter>
__global__ void __launch_bounds__(kWarps * 32) norm_rope_backward_kernel(const __grid_constant__ Args a) {
  using C = RowCfg<T, D>;
  constexpr int E = C::E, W = C::kWords, kAhead = 2;
  __shared__ float sums[kWarps][2][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / C::L, at = lane % C::L * E;
  let_next_start();
  wait_for_previous();
  const long long tokens = static_cast<long long>(a.B) * a.S;
  Turn<T, D, kInter> turn;
  turn.place(a, lane);
  float dw[2][E];
#pragma unroll
  for (int e = 0; e < E; ++e) dw[0][e] = dw[1][e] = 0.f;
  for (long long token = static_cast<long long>(blockIdx.x) * kWarps + warp; token < tokens;
       token += static_cast<long long>(gridDim.x) * kWarps) {
    const int b = static_cast<int>(token / a.S), t = static_cast<int>(token - static_cast<long long>(b) * a.S);
    turn.angles(a, lane, a.rot_dim ? row_position(a, b, t) : 0);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int heads = a.heads[side], groups = (heads + C::R - 1) / C::R;
      if (heads == 0) continue;
      const Rows in = a.in[side], dy = a.dy[side], out = a.out[side];
      const bool norm = a.w[side] != nullptr;
      const T* src = reinterpret_cast<const T*>(in.data) + (norm ? b * in.batch + t * in.row + at : 0);
      const T* grad = reinterpret_cast<const T*>(dy.data) + b * dy.batch + t * dy.row + at;
      T* dst = reinterpret_cast<T*>(out.data) + b * out.batch + t * out.row + at;
      float w[E];
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = norm ? weight_at(a.w[side], a.w_f32, at + e, T()) : 1.f;
      for (int g = 0; g < groups; g += kAhead) {
        unsigned ux[kAhead][W], ug[kAhead][W];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int h = (g + i) * C::R + sub;
#pragma unroll
          for (int j = 0; j < W; ++j) ux[i][j] = ug[i][j] = 0;
          if (h < heads) {
            load_words<T, W>(grad + h * dy.head, dy.vec, ug[i]);
            if (norm) load_words<T, W>(src + h * in.head, in.vec, ux[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (g + i >= groups) break;
          const int h = (g + i) * C::R + sub;
          float x[E], y[E], gr[E];
          unpack<T, E>(ug[i], y);
          turn.other(ug[i], y, gr);
#pragma unroll
          for (int e = 0; e < E; ++e) gr[e] = turn.turns ? fmaf(y[e], turn.c[e], -gr[e] * turn.s[e]) : y[e];
          if (norm) {
            unpack<T, E>(ux[i], x);
            float sq = 0.f, dot = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
              sq = fmaf(x[e], x[e], sq);
              dot = fmaf(gr[e] * w[e], x[e], dot);
            }
            sq = row_sum<C::L>(sq);
            dot = row_sum<C::L>(dot);
            const float r = rsqrtf(sq * (1.f / D) + a.eps);
            const float back = dot * (1.f / D) * r * r;
#pragma unroll
            for (int e = 0; e < E; ++e) {
              dw[side][e] = fmaf(gr[e], x[e] * r, dw[side][e]);
              gr[e] = r * (gr[e] * w[e] - x[e] * back);
            }
          }
          pack<T, E>(gr, ug[i]);
          if (h < heads) store_words<T, W>(dst + h * out.head, out.vec, ug[i]);
        }
      }
    }
  }
  if (a.part == nullptr) return;
  // the rows of the warp, then the warps of the block
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float v = dw[side][e];
#pragma unroll
      for (int i = C::L; i < 32; i *= 2) v += __shfl_xor_sync(0xffffffffu, v, i);
      if (sub == 0) sums[warp][side][at + e] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kWarps * 32) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += sums[w][i / D][i % D];
    a.part[static_cast<size_t>(blockIdx.x) * 2 * D + i] = v;
  }
}

// The blocks' sums into the weights' gradients: 32 columns a block, eight slices of the list each.
__global__ void __launch_bounds__(256) weight_grad_kernel(const float* part, int blocks, int D, float* dq, float* dk) {
  __shared__ float sums[8][32];
  const int col = threadIdx.x & 31, slice = threadIdx.x >> 5, i = blockIdx.x * 32 + col;
  let_next_start();
  wait_for_previous();
  float v = 0.f;
#pragma unroll 8
  for (int n = slice; n < blocks; n += 8) v += part[static_cast<size_t>(n) * 2 * D + i];
  sums[slice][col] = v;
  __syncthreads();
  if (slice != 0) return;
  float all = 0.f;
#pragma unroll
  for (int s = 0; s < 8; ++s) all += sums[s][col];
  float* const out = i < D ? dq : dk;
  if (out) out[i % D] = all;
}

// ---- host side ----------------------------------------------------------------------

constexpr int kBackwardPerSm = 4;  // blocks of the backward pass on an SM

bool aligned_rows(const ra_rows& r, int es, int batch, int heads, int rows) {
  unsigned long long all = reinterpret_cast<uintptr_t>(r.data);
  if (batch > 1) all |= static_cast<unsigned long long>(r.batch_stride) * es;
  if (heads > 1) all |= static_cast<unsigned long long>(r.head_stride) * es;
  if (rows > 1) all |= static_cast<unsigned long long>(r.row_stride) * es;
  return (all & 15u) == 0;
}

Rows make_rows(const ra_rows& r, int es, int batch, int heads, int rows) {
  return {static_cast<char*>(r.data), r.batch_stride, r.head_stride, r.row_stride, aligned_rows(r, es, batch, heads, rows)};
}

// What the three entry points check alike; fills everything of `a` but rows and pages. `segments`: positions may come from
// how->segmap.
int common_args(Args* a, int* inter, const char* what, int dtype, int batch, int seq, int head_dim, const ra_norm_rope* how,
                bool segments) {
  RAB_REQUIRE(dtype == RA_F32 || dtype == RA_F16 || dtype == RA_BF16, RA_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  RAB_REQUIRE(batch >= 0 && seq >= 0, RA_ERR_INVALID, "%s: bad shape", what);
  RAB_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256, RA_ERR_UNSUPPORTED,
              "%s: unsupported head_dim=%d (supported: 32, 64, 128, 256)", what, head_dim);
  std::memset(a, 0, sizeof(*a));
  a->B = batch;
  a->S = seq;
  a->map = affine_posmap(0, seq);
  a->pos_stride = 1;
  *inter = 0;
  if (!how) return RA_OK;
  RAB_REQUIRE(!(how->q_weight || how->k_weight) || how->weight_dtype == dtype || how->weight_dtype == RA_F32, RA_ERR_INVALID,
              "%s: weights are of the rows' dtype or fp32", what);
  RAB_REQUIRE(how->eps >= 0.f, RA_ERR_INVALID, "%s: eps must be >= 0", what);
  a->w[0] = how->q_weight;
  a->w[1] = how->k_weight;
  a->w_f32 = how->weight_dtype == RA_F32;
  a->eps = how->eps;
  if (!how->rope) return RA_OK;
  const int rot = how->rope->rot_dim;
  RAB_REQUIRE(rot >= 16 && rot % 16 == 0 && rot <= head_dim, RA_ERR_INVALID,
              "%s: rot_dim=%d (a multiple of 16, at most head_dim=%d)", what, rot, head_dim);
  a->rot_dim = rot;
  *inter = how->rope->interleaved != 0;
  std::memcpy(a->turns, how->rope->turns, sizeof(a->turns));
  if (how->positions) {
    RAB_REQUIRE(batch <= 1 || how->pos_batch_stride >= 0, RA_ERR_INVALID, "%s: bad stride of positions", what);
    a->positions = how->positions;
    a->pos_batch = how->pos_batch_stride;
  } else if (segments) {
    RAB_REQUIRE(how->segmap != nullptr, RA_ERR_INVALID, "%s: a rotation needs positions or a segment map", what);
    RAB_REQUIRE(how->pos_stride >= 1, RA_ERR_INVALID, "%s: pos_stride must be >= 1", what);
    RAB_REQUIRE(how->segmap->n_seg >= 1 && how->segmap->n_seg <= RA_MAX_SEG &&
                    (seq == 0 || static_cast<long long>(how->segmap->n_seg) * how->segmap->seg_len == seq),
                RA_ERR_INVALID, "%s: n_seg * seg_len must equal the sequence length", what);
    a->map = make_posmap(*how->segmap);
    a->pos_stride = how->pos_stride;
  }
  return RA_OK;
}

// Calls f with the element type, head_dim and the pairing as template arguments.
template <typename F>
int dispatch(int dtype, int head_dim, int inter, F f) {
  auto by_inter = [&](auto t, auto d) {
    return inter ? f(t, d, std::integral_constant<bool, true>()) : f(t, d, std::integral_constant<bool, false>());
  };
  auto by_dim = [&](auto t) {
    if (head_dim == 32) return by_inter(t, std::integral_constant<int, 32>());
    if (head_dim == 64) return by_inter(t, std::integral_constant<int, 64>());
    if (head_dim == 128) return by_inter(t, std::integral_constant<int, 128>());
    return by_inter(t, std::integral_constant<int, 256>());
  };
  if (dtype == RA_F32) return by_dim(float());
  if (dtype == RA_F16) return by_dim(__half());
  return by_dim(__nv_bfloat16());
}

// How many groups of rows a warp takes of a token: all of them where there are tokens enough to fill the SMs with warps, since
// the angles are then worked out once a token, fewer where there are not.
int groups_per_warp(long long tokens, int groups) {
  const long long warps = 16ll * sm_count();
  const long long chunks = tokens >= warps ? 1 : (warps + tokens - 1) / tokens;
  return static_cast<int>((groups + chunks - 1) / chunks);
}

template <bool kPaged>
int launch_forward(int dtype, int head_dim, int inter, const Args& a, cudaStream_t stream) {
  return dispatch(dtype, head_dim, inter, [&](auto t, auto d, auto i) -> int {
    using C = RowCfg<decltype(t), d()>;
    int groups = 0;
    for (int side = 0; side < 3; ++side) groups += (a.heads[side] + C::R - 1) / C::R;
    const long long tokens = static_cast<long long>(a.B) * a.S;
    if (tokens == 0 || groups == 0) return RA_OK;
    const int per = groups_per_warp(tokens, groups);
    const long long total = tokens * ((groups + per - 1) / per), blocks = (total + kWarps - 1) / kWarps;
    RAB_REQUIRE(blocks < (1ll << 31), RA_ERR_INVALID, "norm and rotation: too many rows");
    RAB_CUDA(launch_overlapped(norm_rope_kernel<decltype(t), d(), i(), kPaged>, dim3(static_cast<unsigned>(blocks)),
                               dim3(kWarps * 32), 0, stream, a, total, per));
    return RA_OK;
  });
}

int pair_turns(ra_rope* rope, int rot_dim, int interleaved, const char* what) {
  RAB_REQUIRE(rope != nullptr, RA_ERR_INVALID, "%s: null argument", what);
  RAB_REQUIRE(rot_dim >= 16 && rot_dim % 16 == 0 && rot_dim <= 2 * RA_ROPE_MAX_PAIRS, RA_ERR_INVALID,
              "%s: rot_dim=%d (a multiple of 16, up to %d)", what, rot_dim, 2 * RA_ROPE_MAX_PAIRS);
  std::memset(rope, 0, sizeof(*rope));
  rope->rot_dim = rot_dim;
  rope->interleaved = interleaved != 0;
  return RA_OK;
}

unsigned long long turn_part(long double freq) {
  constexpr long double kTwoPi = 6.283185307179586476925286766559005768L;
  long double t = std::fabs(freq) / kTwoPi;
  t = std::floor((t - std::floor(t)) * 18446744073709551616.0L + 0.5L);
  const unsigned long long turns = t >= 18446744073709551616.0L ? 0ull : static_cast<unsigned long long>(t);
  return freq < 0 ? 0ull - turns : turns;
}

}  // namespace
}  // namespace rab

using namespace rab;

extern "C" {

int ra_rope_init(ra_rope* rope, int rot_dim, int interleaved, double base, double scale) {
  const int rc = pair_turns(rope, rot_dim, interleaved, "ra_rope_init");
  if (rc != RA_OK) return rc;
  RAB_REQUIRE(base > 0 && std::isfinite(base) && std::isfinite(scale), RA_ERR_INVALID, "ra_rope_init: bad base or scale");
  for (int i = 0; i < rot_dim / 2; ++i)
    rope->turns[i] = turn_part(std::pow(static_cast<long double>(base), -2.0L * i / rot_dim) * scale);
  return RA_OK;
}

int ra_rope_init_freqs(ra_rope* rope, int rot_dim, int interleaved, const double* freqs) {
  RAB_REQUIRE(freqs != nullptr, RA_ERR_INVALID, "ra_rope_init_freqs: null argument");
  const int rc = pair_turns(rope, rot_dim, interleaved, "ra_rope_init_freqs");
  if (rc != RA_OK) return rc;
  for (int i = 0; i < rot_dim / 2; ++i) {
    RAB_REQUIRE(std::isfinite(freqs[i]), RA_ERR_INVALID, "ra_rope_init_freqs: frequency %d is not finite", i);
    rope->turns[i] = turn_part(freqs[i]);
  }
  return RA_OK;
}

int ra_qk_norm_rope(int dtype, const ra_rows* q, const ra_rows* k, const ra_rows* q_out, const ra_rows* k_out,
                    const ra_shape* shape, const ra_norm_rope* how, ra_stream stream) {
  RAB_REQUIRE(shape && how, RA_ERR_INVALID, "qk_norm_rope: null argument");
  RAB_REQUIRE(shape->seq_q == shape->seq_k, RA_ERR_INVALID, "qk_norm_rope: queries and keys are of the same tokens");
  Args a;
  int inter = 0;
  const int rc = common_args(&a, &inter, "qk_norm_rope", dtype, shape->batch, shape->seq_q, shape->head_dim, how, true);
  if (rc != RA_OK) return rc;
  const ra_rows* in[2] = {q, k};
  const ra_rows* out[2] = {q_out, k_out};
  const int heads[2] = {shape->heads, kv_heads_of(*shape)};
  const bool empty = shape->batch == 0 || shape->seq_q == 0;
  for (int side = 0; side < 2; ++side) {
    RAB_REQUIRE(!in[side] == !out[side], RA_ERR_INVALID, "qk_norm_rope: rows without a result, or a result without rows");
    if (!in[side]) continue;
    RAB_REQUIRE(heads[side] > 0, RA_ERR_INVALID, "qk_norm_rope: bad heads");
    RAB_REQUIRE(empty || (in[side]->data && out[side]->data), RA_ERR_INVALID, "qk_norm_rope: null argument");
    a.heads[side] = heads[side];
    const int es = dtype == RA_F32 ? 4 : 2;
    a.in[side] = make_rows(*in[side], es, a.B, heads[side], a.S);
    a.out[side] = make_rows(*out[side], es, a.B, heads[side], a.S);
  }
  return launch_forward<false>(dtype, shape->head_dim, inter, a, static_cast<cudaStream_t>(stream));
}

size_t ra_qk_norm_rope_backward_workspace_bytes(int head_dim) {
  return head_dim > 0 ? static_cast<size_t>(kBackwardPerSm) * sm_count() * 2 * head_dim * sizeof(float) : 0;
}

int ra_qk_norm_rope_backward(int dtype, const ra_rows* q, const ra_rows* k, const ra_rows* dq_out, const ra_rows* dk_out,
                             const ra_rows* dq, const ra_rows* dk, float* dq_weight, float* dk_weight,
                             const ra_shape* shape, const ra_norm_rope* how, void* workspace, size_t workspace_bytes,
                             ra_stream stream_) {
  const char* const what = "qk_norm_rope_backward";
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  RAB_REQUIRE(shape && how, RA_ERR_INVALID, "%s: null argument", what);
  RAB_REQUIRE(shape->seq_q == shape->seq_k, RA_ERR_INVALID, "%s: queries and keys are of the same tokens", what);
  Args a;
  int inter = 0;
  const int rc = common_args(&a, &inter, what, dtype, shape->batch, shape->seq_q, shape->head_dim, how, true);
  if (rc != RA_OK) return rc;
  const ra_rows *in[2] = {q, k}, *grad[2] = {dq_out, dk_out}, *out[2] = {dq, dk};
  float* const dw[2] = {dq_weight, dk_weight};
  const int heads[2] = {shape->heads, kv_heads_of(*shape)};
  const bool empty = shape->batch == 0 || shape->seq_q == 0;
  for (int side = 0; side < 2; ++side) {
    RAB_REQUIRE(!grad[side] == !out[side], RA_ERR_INVALID, "%s: a gradient of the result without one of the rows, or the other way round", what);
    RAB_REQUIRE(!dw[side] || (a.w[side] && grad[side]), RA_ERR_INVALID, "%s: a gradient of a weight that there is not", what);
    if (!grad[side]) continue;
    RAB_REQUIRE(heads[side] > 0, RA_ERR_INVALID, "%s: bad heads", what);
    RAB_REQUIRE(!a.w[side] || in[side], RA_ERR_INVALID, "%s: the norm's gradient needs the rows", what);
    RAB_REQUIRE(empty || (grad[side]->data && out[side]->data && (!a.w[side] || in[side]->data)), RA_ERR_INVALID,
                "%s: null argument", what);
    a.heads[side] = heads[side];
    const int es = dtype == RA_F32 ? 4 : 2;
    if (a.w[side]) a.in[side] = make_rows(*in[side], es, a.B, heads[side], a.S);
    a.dy[side] = make_rows(*grad[side], es, a.B, heads[side], a.S);
    a.out[side] = make_rows(*out[side], es, a.B, heads[side], a.S);
  }
  const bool want = dq_weight || dk_weight;
  RAB_REQUIRE(!want || (workspace && workspace_bytes >= ra_qk_norm_rope_backward_workspace_bytes(shape->head_dim)),
              RA_ERR_OVERFLOW, "%s: workspace too small", what);
  const long long tokens = static_cast<long long>(a.B) * a.S;
  const long long need = (tokens + kWarps - 1) / kWarps;
  const int blocks = static_cast<int>(std::min<long long>(need, static_cast<long long>(kBackwardPerSm) * sm_count()));
  a.part = want ? static_cast<float*>(workspace) : nullptr;
  if (blocks > 0) {
    const int rc2 = dispatch(dtype, shape->head_dim, inter, [&](auto t, auto d, auto i) -> int {
      RAB_CUDA(launch_overlapped(norm_rope_backward_kernel<decltype(t), d(), i()>, dim3(static_cast<unsigned>(blocks)),
                                 dim3(kWarps * 32), 0, stream, a));
      return RA_OK;
    });
    if (rc2 != RA_OK) return rc2;
  }
  if (want)  // (no tokens: zeros)
    RAB_CUDA(launch_overlapped(weight_grad_kernel, dim3(static_cast<unsigned>(2 * shape->head_dim / 32)), dim3(256), 0, stream,
                               a.part, blocks, shape->head_dim, dq_weight, dk_weight));
  return RA_OK;
}

// (the addressing alone, on a page table in host memory)
long long ra_debug_paged_row(const int* table, int max_pages, int num_pages, int page_size, int kv_heads, long long slot) {
  return paged_row(table, max_pages, num_pages, page_shift(page_size), kv_heads, slot);
}

int ra_paged_append(const ra_paged_kv* cache, const ra_rows* k, const ra_rows* v, int rows, const int* counts, const ra_rows* q,
                    const ra_rows* q_out, int heads, const ra_norm_rope* how, ra_stream stream) {
  const char* const what = "paged_append";
  RAB_REQUIRE(cache && k && v, RA_ERR_INVALID, "%s: null argument", what);
  Args a;
  int inter = 0;
  int rc = common_args(&a, &inter, what, cache->dtype, cache->batch, rows, cache->head_dim, how, false);
  if (rc == RA_OK) rc = check_paged(*cache, what);
  if (rc != RA_OK) return rc;
  RAB_REQUIRE(!q == !q_out && (!q || heads > 0), RA_ERR_INVALID, "%s: queries without a result, or a result without queries", what);
  if (a.B == 0 || a.S == 0) return RA_OK;
  RAB_REQUIRE(k->data && v->data && (!q || (q->data && q_out->data)), RA_ERR_INVALID, "%s: null argument", what);
  const int es = cache->dtype == RA_F32 ? 4 : 2;
  a.heads[1] = a.heads[2] = cache->kv_heads;
  a.in[1] = make_rows(*k, es, a.B, cache->kv_heads, a.S);
  a.in[2] = make_rows(*v, es, a.B, cache->kv_heads, a.S);
  a.out[1] = {static_cast<char*>(cache->k), 0, 0, 0, 1};
  a.out[2] = {static_cast<char*>(cache->v), 0, 0, 0, 1};
  if (q) {
    a.heads[0] = heads;
    a.in[0] = make_rows(*q, es, a.B, heads, a.S);
    a.out[0] = make_rows(*q_out, es, a.B, heads, a.S);
  }
  a.lens = cache->lens;
  a.counts = counts;
  a.table = cache->page_table;
  a.table_stride = cache->table_stride;
  a.num_pages = cache->num_pages;
  a.max_pages = cache->max_pages;
  a.page_shift = page_shift(cache->page_size);
  return launch_forward<true>(cache->dtype, cache->head_dim, inter, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
