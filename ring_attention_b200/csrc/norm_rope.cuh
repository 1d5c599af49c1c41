// Rows of queries and keys on their way into attention, what norm_rope.cu (norms and position rotation, rows into a paged cache) and
// append_4bit.cu (rows into a paged cache in 4 bits) share: a lane's pieces of a row and how they turn, the forward kernel, and the
// checks of the arguments. norm_rope.cu has the mathematics and what bounds it.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace rab {

namespace {

constexpr int kWarps = 8;
constexpr int kBackwardBlocks = 2;  // of the backward pass, to an SM

// Two pieces of P elements (kBytes) of a row to a lane, L lanes to a row, R rows to a warp.
template <typename T, int D, int kBytes>
struct RowCfg {
  static constexpr int W = kBytes / 4, P = kBytes / static_cast<int>(sizeof(T)), E = 2 * P;
  static constexpr int L = D / E, R = 32 / L;
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
template <typename T, int P, int W>
__device__ inline void unpack(const unsigned (&u)[W], float2 (&x)[P / 2]) {
#pragma unroll
  for (int i = 0; i < P / 2; ++i) {
    if constexpr (sizeof(T) == 4) x[i] = make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
    else x[i] = unpack2<T>(u[i]);
  }
}
// two elements an instruction
__device__ inline float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<unsigned long long*>(&d))
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return d;
}
__device__ inline float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<unsigned long long*>(&d))
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
  return d;
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
template <typename T, int P, int W>
__device__ inline void pack(const float2 (&x)[P / 2], unsigned (&u)[W]) {
#pragma unroll
  for (int i = 0; i < P / 2; ++i) {
    if constexpr (sizeof(T) == 4) u[2 * i] = __float_as_uint(x[i].x), u[2 * i + 1] = __float_as_uint(x[i].y);
    else u[i] = pack2<T>(x[i].x, x[i].y);
  }
}

// A piece of a row: at once, or (`vec` false: some row is not 16-byte aligned) an element at a time.
template <typename T, int W>
__device__ inline void load_piece(const T* p, bool vec, unsigned (&u)[W]) {
  if (vec && W == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    u[0] = v.x, u[1] = v.y, u[W - 2] = v.z, u[W - 1] = v.w;
  } else if (vec) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    u[0] = v.x, u[1] = v.y;
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
__device__ inline void store_piece(T* p, bool vec, const unsigned (&u)[W]) {
  if (vec && W == 4) {
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[W - 2], u[W - 1]);
  } else if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
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

// Bytes of a piece. The backward pass has a lane's share of the weights' gradients in registers beside two rows, and takes half as
// much of a 16-bit row.
constexpr int kForwardBytes = 16;
template <typename T>
constexpr int kBackwardBytes = sizeof(T) == 2 ? 8 : 16;

struct Rows {
  char* data;
  long long batch, head, row;  // strides in elements
  int vec;                     // every row is 16-byte aligned
};

struct Args {
  Rows in[3], dy[2], out[3];  // q, k, v (v and a cache's k_out, v_out: see paged below)
  int heads[3];               // 0: that side is absent
  unsigned S;
  const void* w[2];
  int w_f32, w_vec;  // fp32 or of the rows' type; both 16-byte aligned
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
  float scale[3];  // rows in 4 bits: the factor of side 1's and of side 2's scales
  float* part;  // backward: partial sums of the weights' gradients, [block][2][D]
  unsigned long long turns[RA_ROPE_MAX_PAIRS];
};

// P weights from element `at` on.
template <typename T, int P>
__device__ inline void load_weights(const void* w, int w_f32, int vec, int at, float2 (&x)[P / 2]) {
  if (sizeof(T) == 2 && w_f32) {
    unsigned u[4];
#pragma unroll
    for (int i = 0; i < P / 4; ++i) {
      load_piece<float, 4>(static_cast<const float*>(w) + at + 4 * i, vec, u);
      x[2 * i] = make_float2(__uint_as_float(u[0]), __uint_as_float(u[1]));
      x[2 * i + 1] = make_float2(__uint_as_float(u[2]), __uint_as_float(u[3]));
    }
  } else {
    unsigned u[P * sizeof(T) / 4];
    load_piece<T>(static_cast<const T*>(w) + at, vec, u);
    unpack<T, P>(u, x);
  }
}

__device__ inline long long row_position(const Args& a, int b, int s) {
  if (a.positions) return a.positions[b * a.pos_batch + s];
  if (a.lens) return static_cast<long long>(a.lens[b]) + s;
  const int seg = static_cast<int>(static_cast<unsigned>(s) / static_cast<unsigned>(a.map.seg_len));
  return a.map.base[seg] + static_cast<long long>(s - seg * a.map.seg_len) * a.pos_stride;
}

// A lane's two pieces of a row and how they turn: y[q] = x[q] (cos) + other(x)[q] (signed sin), q = 0, 1, where other exchanges
// what turns into one another: the pieces, or (kInter) neighbours. Behind rot_dim nothing turns: cos 1, sin 0, and nothing other,
// whatever the elements hold.
template <typename T, int D, bool kInter, int kBytes>
struct Turn {
  using C = RowCfg<T, D, kBytes>;
  static constexpr int P = C::P;
  int at[2];   // first element of each piece
  bool turns;
  float2 c[P / 2], s[P / 2];  // of the lane's P pairs
  __device__ inline void place(const Args& a, int lane) {
    const int l = lane % C::L;
    turns = l * C::E < a.rot_dim;
    at[0] = !kInter && turns ? l * P : l * C::E;
    at[1] = at[0] + (!kInter && turns ? a.rot_dim / 2 : P);
  }
  __device__ inline void angles(const unsigned long long* turns_of, int lane, long long pos) {
#pragma unroll
    for (int e = 0; e < P / 2; ++e) c[e] = make_float2(1.f, 1.f), s[e] = make_float2(0.f, 0.f);
    if (!turns) return;
    // (the angle in half turns, from the upper word of its place in the turn: off by 2^-25 of a half turn at most)
    auto angle = [&](int pair, float* si, float* co) {
      const unsigned long long t = static_cast<unsigned long long>(pos) * turns_of[pair];
      sincospif(static_cast<float>(static_cast<int>(t >> 32)) * 4.656612873077393e-10f, si, co);
    };
    const int pair = lane % C::L * P;
#pragma unroll
    for (int e = 0; e < P / 2; ++e) {
      angle(pair + 2 * e, &s[e].x, &c[e].x);
      angle(pair + 2 * e + 1, &s[e].y, &c[e].y);
    }
  }
  // cos and signed sin of element pair e of piece q
  __device__ inline float2 cos_of(int q, int e) const {
    if constexpr (!kInter) return c[e];
    const float v = e % 2 ? c[q * (P / 4) + e / 2].y : c[q * (P / 4) + e / 2].x;
    return make_float2(v, v);
  }
  __device__ inline float2 sin_back(int q, int e) const {  // of the turn back
    if constexpr (!kInter) return q == 0 ? s[e] : make_float2(-s[e].x, -s[e].y);
    const float v = e % 2 ? s[q * (P / 4) + e / 2].y : s[q * (P / 4) + e / 2].x;
    return make_float2(v, -v);
  }
  __device__ inline float2 sin_of(int q, int e) const {
    if constexpr (!kInter) return q == 0 ? make_float2(-s[e].x, -s[e].y) : s[e];
    const float v = e % 2 ? s[q * (P / 4) + e / 2].y : s[q * (P / 4) + e / 2].x;
    return make_float2(-v, v);
  }
  // (kAll: all of the row turns)
  template <bool kAll>
  __device__ inline float2 other(const float2 (&x)[2][P / 2], int q, int e) const {
    const float2 o = kInter ? make_float2(x[q][e].y, x[q][e].x) : x[1 - q][e];
    return kAll || turns ? o : make_float2(0.f, 0.f);
  }
};

// The rotation's table into shared memory (from the launch's parameters, where lanes that ask for different entries wait for one
// another).
__device__ inline void load_turns(const Args& a, unsigned long long* turns_of) {
  for (int i = threadIdx.x; i < a.rot_dim / 2; i += kWarps * 32) turns_of[i] = a.turns[i];
  __syncthreads();
}

template <int L>
__device__ inline float row_sum(float v) {
#pragma unroll
  for (int i = L / 2; i > 0; i /= 2) v += __shfl_xor_sync(0xffffffffu, v, i);
  return v;
}

// ---- rows in 4 bits -----------------------------------------------------------------

__device__ inline float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 16 elements of a 16-bit row as their codes and their scale's byte. The scale is the nearest e4m3 to their largest magnitude / 6 (of
// 448 at most; NaN if one of them is), in units of `factor`, a power of two; a code is the nearest e2m1 to its element / scale, of two
// equally near ones the even. An element / scale is worked out as a product with the reciprocal, off by less than 2^-22 of it, and then
// rounded to 16 bits: the middle between two codes has 3 bits and an element 11 at most, so a quotient that is not such a middle is
// 2^-11 and more from it, and one that is comes out as it.
template <typename T>
__device__ inline void to_4bit(const unsigned (&u)[8], float factor, uint2* codes, unsigned* scale) {
  float2 x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = unpack2<T>(u[i]);
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m[i] = max_nan(max_nan(fabsf(x[2 * i].x), fabsf(x[2 * i].y)), max_nan(fabsf(x[2 * i + 1].x), fabsf(x[2 * i + 1].y)));
  const float most = max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3]));
  const float want = __fdiv_rn(most * __frcp_rn(factor), 6.f);
  unsigned short two;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.f), "f"(want));
  *scale = two & 0xffu;
  unsigned half;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(half) : "h"(two));
  const float step = __half2float(__ushort_as_half(static_cast<unsigned short>(half))) * factor;
  const float inv = step > 0.f ? __frcp_rn(step) : 0.f;
  auto quotient = [&](float v) { return __uint_as_float((__float_as_uint(v * inv) + 0x80u) & 0xffffff00u); };
  unsigned w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(w[i])
        : "f"(quotient(x[4 * i].x)), "f"(quotient(x[4 * i].y)), "f"(quotient(x[4 * i + 1].x)), "f"(quotient(x[4 * i + 1].y)),
          "f"(quotient(x[4 * i + 2].x)), "f"(quotient(x[4 * i + 2].y)), "f"(quotient(x[4 * i + 3].x)), "f"(quotient(x[4 * i + 3].y)));
  *codes = make_uint2(w[0], w[1]);
}

// A warp has the rows of kAhead heads on their way; two blocks of eight warps to an SM leave a thread 128 registers. us a pass
// (32768 tokens of 40 heads of 128, bf16; by one token a warp): 117, with three heads 124, three blocks and two heads 122, 8-byte pieces
// 122.
// A warp takes R of the `total` tokens, a row's lanes one of them, and `per` heads of each, from the list of q's heads, then k's,
// then v's. kFour: the cache holds rows in 4 bits. A row is then worked out and rounded as for a cache in 16 bits, and a lane makes the
// codes of one block of 16 elements: of its two pieces, or, where those are half a rotation apart, of what lies side by side once the
// lanes of the row have exchanged their pieces through shared memory.
template <typename T, int D, bool kInter, bool kPaged, bool kFour = false>
__global__ void __launch_bounds__(kWarps * 32, 2) norm_rope_kernel(const __grid_constant__ Args a, unsigned total, int per) {
  using C = RowCfg<T, D, kForwardBytes>;
  constexpr int P = C::P, kAhead = 4;
  const int lane = threadIdx.x & 31, sub = lane / C::L;
  __shared__ unsigned long long turns_of[RA_ROPE_MAX_PAIRS];
  __shared__ uint4 pieces[kFour ? kWarps : 1][kFour ? 64 : 1];
  const unsigned token0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * C::R;
  let_next_start();
  load_turns(a, turns_of);
  wait_for_previous();
  if (token0 >= total) return;
  const bool there = token0 + sub < total;  // (lanes without a token read the last one's rows, and store nothing)
  const unsigned token = min(token0 + sub, total - 1);
  int b = static_cast<int>(token / a.S), t = static_cast<int>(token - static_cast<unsigned>(b) * a.S);
  bool mine = there;
  long long place = -1;  // paged: row of the cache's first head that takes the token's K and V
  if constexpr (kPaged) {
    if (a.counts) mine = mine && t < a.counts[b];
    const unsigned some = __ballot_sync(0xffffffffu, mine);
    if (some == 0) return;
    // (rows behind a count are not read either)
    const int from = __ffs(static_cast<int>(some)) - 1;
    const int b_from = __shfl_sync(0xffffffffu, b, from), t_from = __shfl_sync(0xffffffffu, t, from);
    if (!mine) b = b_from, t = t_from;
    else place = paged_row(a.table + b * a.table_stride, a.max_pages, a.num_pages, a.page_shift, a.heads[1],
                           static_cast<long long>(a.lens[b]) + t);
  }
  Turn<T, D, kInter, kForwardBytes> turn;
  turn.place(a, lane);
  const long long pos = a.rot_dim ? row_position(a, b, t) : 0;
  const int beg = static_cast<int>(blockIdx.y) * per, end = beg + per;
  int first = 0;  // place of a side's first head in the list
  bool turned = false;
#pragma unroll
  for (int side = 0; side < (kPaged ? 3 : 2); ++side) {
    const int lo = max(beg - first, 0), hi = min(end - first, a.heads[side]);
    first += a.heads[side];
    if (lo >= hi) continue;
    const bool to_cache = kPaged && side > 0, store = to_cache ? place >= 0 : mine;
    const Rows in = a.in[side], out = a.out[side];
    const long long out_head = to_cache ? static_cast<long long>(D) << a.page_shift : out.head;
    const T* src = reinterpret_cast<const T*>(in.data) + b * in.batch + t * in.row;
    T* dst = reinterpret_cast<T*>(out.data) + (to_cache ? place * D : b * out.batch + t * out.row) + lo * out_head;
    [[maybe_unused]] unsigned char* four = nullptr;  // first head's rows of the token's page
    [[maybe_unused]] const int four_row = static_cast<int>(place) & ((1 << a.page_shift) - 1);
    if constexpr (kFour) {
      if (to_cache && store)
        four = reinterpret_cast<unsigned char*>(out.data) + ((place >> a.page_shift) + lo << a.page_shift) * four_row_bytes(D);
    }
    unsigned u[kAhead][2][C::W];
    auto load = [&](int g) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (g + i >= hi) break;
        const T* const row = src + (g + i) * in.head;
#pragma unroll
        for (int q = 0; q < 2; ++q) load_piece<T, C::W>(row + turn.at[q], in.vec, u[i][q]);
      }
    };
    load(lo);  // (on their way while the angles are worked out)
    // factors of a lane's elements and of those that turn into them, weights included
    float2 fx[2][P / 2], fp[2][P / 2];
    const bool norm = side < 2 && a.w[side < 2 ? side : 0] != nullptr;
    if (side < 2) {
      if (!turned && a.rot_dim) turn.angles(turns_of, lane, pos);
      if (!turned && !a.rot_dim) {
#pragma unroll
        for (int e = 0; e < P / 2; ++e) turn.c[e] = make_float2(1.f, 1.f), turn.s[e] = make_float2(0.f, 0.f);
      }
      turned = true;
      float2 w[2][P / 2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int e = 0; e < P / 2; ++e) w[q][e] = make_float2(1.f, 1.f);
        if (norm) load_weights<T, P>(a.w[side], a.w_f32, a.w_vec, turn.at[q], w[q]);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < P / 2; ++e) {
          fx[q][e] = mul2(turn.cos_of(q, e), w[q][e]);
          fp[q][e] = mul2(turn.sin_of(q, e), turn.template other<false>(w, q, e));
        }
    }
    auto rows = [&](auto all) {
      constexpr bool kAll = decltype(all)::value;
      for (int g = lo; g < hi; g += kAhead) {
        if (g > lo) load(g);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (g + i >= hi) break;
          if (side < 2) {
            float2 x[2][P / 2], y[P / 2];
            unpack<T, P>(u[i][0], x[0]);
            unpack<T, P>(u[i][1], x[1]);
            float r = 1.f;
            if (norm) {
              float2 sum = mul2(x[0][0], x[0][0]), more = mul2(x[1][0], x[1][0]);
#pragma unroll
              for (int e = 1; e < P / 2; ++e) {
                sum = fma2(x[0][e], x[0][e], sum);
                more = fma2(x[1][e], x[1][e], more);
              }
              r = rsqrtf(row_sum<C::L>((sum.x + sum.y) + (more.x + more.y)) * (1.f / D) + a.eps);
            }
            const float2 r2 = make_float2(r, r);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
              for (int e = 0; e < P / 2; ++e)
                y[e] = mul2(r2, fma2(x[q][e], fx[q][e], mul2(turn.template other<kAll>(x, q, e), fp[q][e])));
              pack<T, P>(y, u[i][q]);
            }
          }
          if constexpr (kFour) {
            if (to_cache) {
              const int block = lane % C::L;
              unsigned e[8];
              if (!kInter && a.rot_dim) {
                uint4* const row = &pieces[threadIdx.x >> 5][2 * (lane - block)];
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 2; ++q) row[turn.at[q] / 8] = make_uint4(u[i][q][0], u[i][q][1], u[i][q][2], u[i][q][3]);
                __syncwarp();
                const uint4 x = row[2 * block], y = row[2 * block + 1];
                e[0] = x.x, e[1] = x.y, e[2] = x.z, e[3] = x.w, e[4] = y.x, e[5] = y.y, e[6] = y.z, e[7] = y.w;
              } else {
#pragma unroll
                for (int q = 0; q < 8; ++q) e[q] = u[i][q / 4][q % 4];
              }
              uint2 codes;
              unsigned scale;
              to_4bit<T>(e, a.scale[side], &codes, &scale);
              if (store) {
                *reinterpret_cast<uint2*>(four + four_row * (D / 2) + ((block / 2) ^ four_turn(four_row, D)) * 16 + block % 2 * 8) = codes;
                four[(D / 2 << a.page_shift) + four_row * (D / 16) + block] = static_cast<unsigned char>(scale);
                four += static_cast<long long>(four_row_bytes(D)) << a.page_shift;
              }
              continue;
            }
          }
          if (store) {
#pragma unroll
            for (int q = 0; q < 2; ++q) store_piece<T, C::W>(dst + turn.at[q], out.vec, u[i][q]);
          }
          dst += out_head;
        }
      }
    };
    if (a.rot_dim == D) rows(std::true_type());
    else rows(std::false_type());
  }
}

// ---- host side ----------------------------------------------------------------------

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

// Rows are read an element at a time where they are not 16-byte aligned, so that elements have to be.
bool whole_elements(const ra_rows* r, int dtype) {
  return !r || (reinterpret_cast<uintptr_t>(r->data) & (dtype == RA_F32 ? 3u : 1u)) == 0;
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
  RAB_REQUIRE(static_cast<long long>(batch) * seq < (1ll << 31), RA_ERR_INVALID, "%s: too many tokens", what);
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
  RAB_REQUIRE(((reinterpret_cast<uintptr_t>(how->q_weight) | reinterpret_cast<uintptr_t>(how->k_weight)) & (a->w_f32 ? 3u : 1u)) == 0 &&
                  (reinterpret_cast<uintptr_t>(how->positions) & 3u) == 0,
              RA_ERR_INVALID, "%s: weights or positions are not aligned to their elements", what);
  a->w_vec = ((reinterpret_cast<uintptr_t>(how->q_weight) | reinterpret_cast<uintptr_t>(how->k_weight)) & 15u) == 0;
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

// Calls f with the element type (k32: fp32 among them), head_dim and the pairing as template arguments.
template <bool k32 = true, typename F>
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
  if constexpr (k32) {
    if (dtype == RA_F32) return by_dim(float());
  }
  if (dtype == RA_F16) return by_dim(__half());
  return by_dim(__nv_bfloat16());
}

// How many heads of its tokens a warp takes, of `heads`, where `groups` warps have the tokens: for the least time of as many rounds
// as the warps that the SMs hold at once need, where a warp costs its heads' rows and kAngles rows for its tokens' angles. us: 32768
// tokens of 40 heads with 40 / 20 (so) / 10 heads a warp 113 / 109 / 120; 500 tokens with 1 / 2 / 3 (so) 8.4 / 6.7 / 5.0; backward of
// 2 x 1531 tokens of 16 heads of 64 in fp32 with 1 / 3 / 6 (so) 18.0 / 13.8 / 13.3.
int heads_per_warp(long long groups, int heads) {
  constexpr int kAngles = 4;
  const long long warps = 16ll * sm_count();
  if (groups * heads <= warps) return 1;
  const int most = static_cast<int>(std::min<long long>(heads, 2 * warps / groups + 2));
  int best = heads;
  long long least = -1;
  for (int chunks = 1; chunks <= most; ++chunks) {
    const int per = (heads + chunks - 1) / chunks;
    const long long cost = (groups * ((heads + per - 1) / per) + warps - 1) / warps * (kAngles + per);
    if (least < 0 || cost < least) least = cost, best = per;
  }
  return best;
}

template <bool kPaged, bool kFour = false>
int launch_forward(int dtype, int head_dim, int inter, const Args& a, unsigned tokens, cudaStream_t stream) {
  return dispatch<!kFour>(dtype, head_dim, inter, [&](auto t, auto d, auto i) -> int {
    using C = RowCfg<decltype(t), d(), kForwardBytes>;
    const int heads = a.heads[0] + a.heads[1] + a.heads[2];
    if (tokens == 0 || heads == 0) return RA_OK;
    const unsigned groups = (tokens + C::R - 1) / C::R;
    const int per = heads_per_warp(groups, heads);
    RAB_CUDA(launch_overlapped(norm_rope_kernel<decltype(t), d(), i(), kPaged, kFour>,
                               dim3((groups + kWarps - 1) / kWarps, static_cast<unsigned>((heads + per - 1) / per)), dim3(kWarps * 32), 0, stream, a, tokens, per));
    return RA_OK;
  });
}

template <typename T>
int launch_plain_4bit(int head_dim, const Args& a, unsigned tokens, cudaStream_t stream);  // append_4bit.cu

// Rows of k, v and q of new tokens to a paged cache and q_out (see ra_paged_append, ra_paged_append_4bit).
template <bool kFour>
int append_rows(const char* what, const ra_paged_kv* cache, const ra_rows* k, const ra_rows* v, int rows, const int* counts,
                const ra_rows* q, const ra_rows* q_out, int heads, const ra_norm_rope* how, float k_scale, float v_scale,
                ra_stream stream) {
  RAB_REQUIRE(cache && k && v, RA_ERR_INVALID, "%s: null argument", what);
  Args a;
  int inter = 0;
  int rc = common_args(&a, &inter, what, cache->dtype, cache->batch, rows, cache->head_dim, how, false);
  if (rc == RA_OK) rc = kFour ? check_paged_4bit(*cache, k_scale, v_scale, what) : check_paged(*cache, what);
  if (rc == RA_OK) rc = check_lists(*cache, what);
  if (rc != RA_OK) return rc;
  RAB_REQUIRE(!q == !q_out && (!q || heads > 0), RA_ERR_INVALID, "%s: queries without a result, or a result without queries", what);
  if (cache->batch == 0 || rows == 0) return RA_OK;
  RAB_REQUIRE(k->data && v->data && (!q || (q->data && q_out->data)), RA_ERR_INVALID, "%s: null argument", what);
  RAB_REQUIRE(whole_elements(k, cache->dtype) && whole_elements(v, cache->dtype) && whole_elements(q, cache->dtype) &&
                  whole_elements(q_out, cache->dtype) && (reinterpret_cast<uintptr_t>(counts) & 3u) == 0,
              RA_ERR_INVALID, "%s: rows or counts are not aligned to their elements", what);
  const int es = cache->dtype == RA_F32 ? 4 : 2;
  a.heads[1] = a.heads[2] = cache->kv_heads;
  a.in[1] = make_rows(*k, es, cache->batch, cache->kv_heads, rows);
  a.in[2] = make_rows(*v, es, cache->batch, cache->kv_heads, rows);
  a.out[1] = {static_cast<char*>(cache->k), 0, 0, 0, 1};
  a.out[2] = {static_cast<char*>(cache->v), 0, 0, 0, 1};
  if (q) {
    a.heads[0] = heads;
    a.in[0] = make_rows(*q, es, cache->batch, heads, rows);
    a.out[0] = make_rows(*q_out, es, cache->batch, heads, rows);
  }
  a.lens = cache->lens;
  a.counts = counts;
  a.table = cache->page_table;
  a.table_stride = cache->table_stride;
  a.num_pages = cache->num_pages;
  a.max_pages = cache->max_pages;
  a.page_shift = page_shift(cache->page_size);
  a.scale[1] = k_scale;
  a.scale[2] = v_scale;
  if constexpr (kFour) {
    if (!q && !a.w[1] && a.rot_dim == 0) {
      const unsigned tokens = static_cast<unsigned>(cache->batch) * a.S;
      return cache->dtype == RA_F16 ? launch_plain_4bit<__half>(cache->head_dim, a, tokens, static_cast<cudaStream_t>(stream))
                                    : launch_plain_4bit<__nv_bfloat16>(cache->head_dim, a, tokens, static_cast<cudaStream_t>(stream));
    }
  }
  return launch_forward<true, kFour>(cache->dtype, cache->head_dim, inter, a, static_cast<unsigned>(cache->batch) * a.S, static_cast<cudaStream_t>(stream));
}

}  // namespace
}  // namespace rab
