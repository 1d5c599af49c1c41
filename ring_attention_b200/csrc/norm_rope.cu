// Rows of queries and keys on their way into attention: the norm of each head's row, the position rotation, and, for a paged
// cache, the place a row goes to; and the backward pass of norm and rotation.
//
//   y = R_p (x r w),  r = (mean(x^2) + eps)^-1/2,  R_p turns pair i by p f_i
//   backward, with g = R_-p dy:  dw = sum over rows of g x r,  dx = r (g w - x r^2 mean(g w x))
//
// All of it is bound by memory: a row comes in once and goes out once. A lane holds two 16-byte pieces of a row, in such a place
// that the elements it turns into one another are its own: with pairs half a row apart, a piece of either half. So 2 to 32
// lanes share a row and nothing crosses lanes but the sum of squares. The row groups of a warp take a token each, one head after the
// other: cos and sin of a token are worked out once for all heads that the warp takes, no lane is idle whatever the heads' number, and
// the rows of a head lie side by side. (With the warp's row groups on heads of one token, each had its angles over again: us a pass, 32768
// tokens of 40 heads of 128 in bf16 117, so 109; 804858 tokens of four heads of 32, backward, 967 and 182.) The angles come from
// fixed point (see ra_rope) and are multiplied by the weights ahead of the rows: a row then costs a sum of squares and three
// multiply-adds an element, two elements an instruction.
// Times in this file are of launches one behind the other in a CUDA graph; calls of less than some 15 us wait for the host otherwise.
#include "norm_rope.cuh"

namespace rab {

namespace {

// The backward pass: a warp walks over units of R tokens and `per` heads of each, `chunks` units to the same tokens, and keeps its
// share of the weights' gradients; the block's sums go to its place in the workspace, in an order that does not depend on timing.
// us a pass (32768 tokens of 32 heads of 128, bf16; 123 at the copy's rate): 167, with three heads on their way 174, six 181 (spills),
// 16-byte pieces 227, three blocks of two heads 229 (both spill); by one token a warp 186, and so with rows through a ring in shared
// memory 184, which cost fp32 (254) 40 more.
template <typename T, int D, bool kInter>
__global__ void __launch_bounds__(kWarps * 32, kBackwardBlocks)
    norm_rope_backward_kernel(const __grid_constant__ Args a, unsigned tokens, unsigned units, unsigned chunks, int per) {
  using C = RowCfg<T, D, kBackwardBytes<T>>;
  constexpr int P = C::P, kAhead = sizeof(T) == 2 ? 4 : 3;
  __shared__ float sums[kWarps][2][D];
  __shared__ unsigned long long turns_of[RA_ROPE_MAX_PAIRS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / C::L;
  let_next_start();
  load_turns(a, turns_of);
  wait_for_previous();
  Turn<T, D, kInter, kBackwardBytes<T>> turn;
  turn.place(a, lane);
  float2 dw[2][2][P / 2];
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int e = 0; e < P / 2; ++e) dw[side][q][e] = make_float2(0.f, 0.f);
#pragma unroll
  for (int e = 0; e < P / 2; ++e) turn.c[e] = make_float2(1.f, 1.f), turn.s[e] = make_float2(0.f, 0.f);
  for (unsigned unit = blockIdx.x * kWarps + warp; unit < units; unit += gridDim.x * kWarps) {
    const unsigned of_tokens = unit / chunks, token0 = of_tokens * C::R;
    const int beg = static_cast<int>(unit - of_tokens * chunks) * per, end = beg + per;
    const bool mine = token0 + sub < tokens;  // (lanes without a token read the last one's rows, store and sum nothing)
    const unsigned token = min(token0 + sub, tokens - 1);
    const int b = static_cast<int>(token / a.S), t = static_cast<int>(token - static_cast<unsigned>(b) * a.S);
    const long long pos = a.rot_dim ? row_position(a, b, t) : 0;
    bool turned = a.rot_dim == 0;
    int first = 0;  // place of a side's first head in the list of q's heads, then k's
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int lo = max(beg - first, 0), hi = min(end - first, a.heads[side]);
      first += a.heads[side];
      if (lo >= hi) continue;
      const Rows in = a.in[side], dy = a.dy[side], out = a.out[side];
      const bool norm = a.w[side] != nullptr;
      const T* src = reinterpret_cast<const T*>(in.data) + (norm ? b * in.batch + t * in.row : 0);
      const T* grad = reinterpret_cast<const T*>(dy.data) + b * dy.batch + t * dy.row;
      T* dst = reinterpret_cast<T*>(out.data) + b * out.batch + t * out.row;
      unsigned ux[kAhead][2][C::W], ug[kAhead][2][C::W];
      auto load = [&](int g) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int h = g + i;
          if (h >= hi) break;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            load_piece<T, C::W>(grad + h * dy.head + turn.at[q], dy.vec, ug[i][q]);
            if (norm) load_piece<T, C::W>(src + h * in.head + turn.at[q], in.vec, ux[i][q]);
          }
        }
      };
      load(lo);  // (on their way while the angles are worked out)
      float2 w[2][P / 2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int e = 0; e < P / 2; ++e) w[q][e] = make_float2(1.f, 1.f);
        if (norm) load_weights<T, P>(a.w[side], a.w_f32, a.w_vec, turn.at[q], w[q]);
      }
      if (!turned) turn.angles(turns_of, lane, pos);
      turned = true;
      auto rows = [&](auto all) {
        constexpr bool kAll = decltype(all)::value;
        for (int g = lo; g < hi; g += kAhead) {
          if (g > lo) load(g);
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const int h = g + i;
            if (h >= hi) break;
            float2 y[2][P / 2], gr[2][P / 2];
            unpack<T, P>(ug[i][0], y[0]);
            unpack<T, P>(ug[i][1], y[1]);
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int e = 0; e < P / 2; ++e)  // (the other way round)
                gr[q][e] = fma2(y[q][e], turn.cos_of(q, e), mul2(turn.template other<kAll>(y, q, e), turn.sin_back(q, e)));
            if (norm) {
              float2 x[2][P / 2], gw[2][P / 2], sq2[2], dot2[2];
              unpack<T, P>(ux[i][0], x[0]);
              unpack<T, P>(ux[i][1], x[1]);
#pragma unroll
              for (int q = 0; q < 2; ++q) {
#pragma unroll
                for (int e = 0; e < P / 2; ++e) {
                  gw[q][e] = mul2(gr[q][e], w[q][e]);
                  sq2[q] = e == 0 ? mul2(x[q][e], x[q][e]) : fma2(x[q][e], x[q][e], sq2[q]);
                  dot2[q] = e == 0 ? mul2(gw[q][e], x[q][e]) : fma2(gw[q][e], x[q][e], dot2[q]);
                }
              }
              const float sq = row_sum<C::L>((sq2[0].x + sq2[0].y) + (sq2[1].x + sq2[1].y));
              const float dot = row_sum<C::L>((dot2[0].x + dot2[0].y) + (dot2[1].x + dot2[1].y));
              const float r = rsqrtf(sq * (1.f / D) + a.eps);
              const float back = -dot * (1.f / D) * r * r;
              const float2 r2 = make_float2(r, r), back2 = make_float2(back, back);
#pragma unroll
              for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int e = 0; e < P / 2; ++e) {
                  if (mine) dw[side][q][e] = fma2(gr[q][e], mul2(x[q][e], r2), dw[side][q][e]);
                  gr[q][e] = mul2(r2, fma2(x[q][e], back2, gw[q][e]));
                }
            }
            if (mine) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                unsigned v[C::W];
                pack<T, P>(gr[q], v);
                store_piece<T, C::W>(dst + h * out.head + turn.at[q], out.vec, v);
              }
            }
          }
        }
      };
      if (a.rot_dim == D) rows(std::true_type());
      else rows(std::false_type());
    }
  }
  if (a.part == nullptr) return;
  // the rows of the warp, then the warps of the block
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int e = 0; e < 2 * P; ++e) {
      float v = e % 2 ? dw[side][e / P][e % P / 2].y : dw[side][e / P][e % P / 2].x;
#pragma unroll
      for (int i = C::L; i < 32; i *= 2) v += __shfl_xor_sync(0xffffffffu, v, i);
      if (sub == 0) sums[warp][side][turn.at[e / P] + e % P] = v;
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
    RAB_REQUIRE(whole_elements(in[side], dtype) && whole_elements(out[side], dtype), RA_ERR_INVALID,
                "qk_norm_rope: rows are not aligned to their elements");
    a.heads[side] = heads[side];
    const int es = dtype == RA_F32 ? 4 : 2;
    a.in[side] = make_rows(*in[side], es, shape->batch, heads[side], a.S);
    a.out[side] = make_rows(*out[side], es, shape->batch, heads[side], a.S);
  }
  return launch_forward<false>(dtype, shape->head_dim, inter, a, static_cast<unsigned>(shape->batch) * a.S, static_cast<cudaStream_t>(stream));
}

size_t ra_qk_norm_rope_backward_workspace_bytes(int head_dim) {
  return head_dim > 0 ? static_cast<size_t>(kBackwardBlocks) * sm_count() * 2 * head_dim * sizeof(float) : 0;
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
    RAB_REQUIRE(whole_elements(in[side], dtype) && whole_elements(grad[side], dtype) && whole_elements(out[side], dtype) &&
                    (reinterpret_cast<uintptr_t>(dw[side]) & 3u) == 0,
                RA_ERR_INVALID, "%s: rows or gradients are not aligned to their elements", what);
    a.heads[side] = heads[side];
    const int es = dtype == RA_F32 ? 4 : 2;
    if (a.w[side]) a.in[side] = make_rows(*in[side], es, shape->batch, heads[side], a.S);
    a.dy[side] = make_rows(*grad[side], es, shape->batch, heads[side], a.S);
    a.out[side] = make_rows(*out[side], es, shape->batch, heads[side], a.S);
  }
  const bool want = dq_weight || dk_weight;
  RAB_REQUIRE(!want || (workspace && workspace_bytes >= ra_qk_norm_rope_backward_workspace_bytes(shape->head_dim) &&
                        (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0),
              RA_ERR_OVERFLOW, "%s: workspace too small or not 16-byte aligned", what);
  const unsigned tokens = static_cast<unsigned>(shape->batch) * a.S;
  a.part = want ? static_cast<float*>(workspace) : nullptr;
  int blocks = 0;
  if (tokens > 0 && a.heads[0] + a.heads[1] > 0) {
    const int rc2 = dispatch(dtype, shape->head_dim, inter, [&](auto t, auto d, auto i) -> int {
      using C = RowCfg<decltype(t), d(), kBackwardBytes<decltype(t)>>;
      const int all = a.heads[0] + a.heads[1];
      const unsigned groups = (tokens + C::R - 1) / C::R;
      const int per = heads_per_warp(groups, all);
      const unsigned chunks = static_cast<unsigned>((all + per - 1) / per), units = groups * chunks;
      blocks = static_cast<int>(std::min<unsigned>((units + kWarps - 1) / kWarps, kBackwardBlocks * sm_count()));
      RAB_CUDA(launch_overlapped(norm_rope_backward_kernel<decltype(t), d(), i()>, dim3(static_cast<unsigned>(blocks)),
                                 dim3(kWarps * 32), 0, stream, a, tokens, units, chunks, per));
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
  return append_rows<false>("paged_append", cache, k, v, rows, counts, q, q_out, heads, how, 1.f, 1.f, stream);
}

}  // extern "C"
