// Rows of K and V to a paged cache in 4 bits, with their norm and rotation and the queries of the same tokens, as paged_append has them
// for a cache in 16 and 32 bits: the same kernel (norm_rope.cuh) with another way out, and one for rows that are only rounded. Bound by
// memory: two bytes an element come in and 9 / 16 of one go out.
#include "norm_rope.cuh"

namespace rab {

namespace {

// Rows that are neither normed nor turned, and no queries: a thread makes the codes of one block of 16 elements of kAhead heads at a time.
// us in a graph, chunks of 2349 to 4099 tokens of four prompts, 8 KV heads of 128 in fp16 (10.3 at the copy's rate): 16, and in the other
// kernel, whose threads hold angles and weights and of which two blocks fit an SM, with K's norm and rotation 24; with those of 32 query
// heads on top, as a step of a server has them, 67 (42.5), where paged_append to a cache in 16 bits takes 61.
constexpr int kPlainThreads = 256, kPlainAhead = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kPlainThreads) plain_4bit_kernel(const __grid_constant__ Args a, unsigned total, int per) {
  constexpr int L = D / 16;
  let_next_start();
  wait_for_previous();
  const unsigned token = blockIdx.x * (kPlainThreads / L) + threadIdx.x / L;  // (threads may be more than 2^32)
  const int block = threadIdx.x % L;
  if (token >= total) return;
  const int b = static_cast<int>(token / a.S), t = static_cast<int>(token - static_cast<unsigned>(b) * a.S);
  if (a.counts && t >= a.counts[b]) return;
  const long long place = paged_row(a.table + b * a.table_stride, a.max_pages, a.num_pages, a.page_shift, a.heads[1],
                                    static_cast<long long>(a.lens[b]) + t);
  if (place < 0) return;
  const int row = static_cast<int>(place) & ((1 << a.page_shift) - 1), kv = a.heads[1];
  const long long page = place >> a.page_shift, piece = static_cast<long long>(four_row_bytes(D)) << a.page_shift;
  const int code_at = row * (D / 2) + ((block / 2) ^ four_turn(row, D)) * 16 + block % 2 * 8;
  const int scale_at = (D / 2 << a.page_shift) + row * (D / 16) + block;
  const int end = min((static_cast<int>(blockIdx.y) + 1) * per, 2 * kv);
  for (int h0 = static_cast<int>(blockIdx.y) * per; h0 < end; h0 += kPlainAhead) {
    unsigned u[kPlainAhead][2][4];
#pragma unroll
    for (int i = 0; i < kPlainAhead; ++i) {
      if (h0 + i >= end) break;
      const int side = h0 + i < kv ? 1 : 2, head = h0 + i - (side - 1) * kv;
      const Rows& in = a.in[side];
      const T* const src = reinterpret_cast<const T*>(in.data) + b * in.batch + t * in.row + head * in.head + block * 16;
      load_piece<T>(src, in.vec, u[i][0]);
      load_piece<T>(src + 8, in.vec, u[i][1]);
    }
#pragma unroll
    for (int i = 0; i < kPlainAhead; ++i) {
      if (h0 + i >= end) break;
      const int side = h0 + i < kv ? 1 : 2, head = h0 + i - (side - 1) * kv;
      unsigned e[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) e[q] = u[i][q / 4][q % 4];
      uint2 codes;
      unsigned scale;
      to_4bit<T>(e, a.scale[side], &codes, &scale);
      unsigned char* const to = reinterpret_cast<unsigned char*>(a.out[side].data) + (page + head) * piece;
      *reinterpret_cast<uint2*>(to + code_at) = codes;
      to[scale_at] = static_cast<unsigned char>(scale);
    }
  }
}

template <typename T>
int launch_plain_4bit(int head_dim, const Args& a, unsigned tokens, cudaStream_t stream) {
  if (tokens == 0) return RA_OK;
  auto go = [&](auto d) -> int {
    constexpr unsigned kTokens = kPlainThreads / (d() / 16);
    const unsigned blocks = (tokens + kTokens - 1) / kTokens;
    // as many heads a thread as loads are on their way, or, where that leaves SMs without a block, one
    const int heads = 2 * a.heads[1];
    const int per = static_cast<long long>(blocks) * ((heads + kPlainAhead - 1) / kPlainAhead) >= 2ll * sm_count() ? kPlainAhead : 1;
    RAB_REQUIRE((heads + per - 1) / per <= 65535, RA_ERR_INVALID, "paged_append_4bit: bad heads");
    RAB_CUDA(launch_overlapped(plain_4bit_kernel<T, d()>, dim3(blocks, static_cast<unsigned>((heads + per - 1) / per)),
                               dim3(kPlainThreads), 0, stream, a, tokens, per));
    return RA_OK;
  };
  if (head_dim == 32) return go(std::integral_constant<int, 32>());
  if (head_dim == 64) return go(std::integral_constant<int, 64>());
  if (head_dim == 128) return go(std::integral_constant<int, 128>());
  return go(std::integral_constant<int, 256>());
}

}  // namespace
}  // namespace rab

using namespace rab;

extern "C" {

int ra_paged_append_4bit(const ra_paged_kv* cache, float k_scale, float v_scale, const ra_rows* k, const ra_rows* v, int rows,
                         const int* counts, const ra_rows* q, const ra_rows* q_out, int heads, const ra_norm_rope* how,
                         ra_stream stream) {
  return append_rows<true>("paged_append_4bit", cache, k, v, rows, counts, q, q_out, heads, how, k_scale, v_scale, stream);
}

}  // extern "C"
