// Attention over packed sequences of unlike lengths, which only the device knows: fp16 / bf16, grouped heads, causal or not, keys as many as
// queries (whole prompts) or more (chunks of prompts behind what is cached of them).
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(q_i . k_j / sqrt(D)),  j <= i + (keys - queries) of the sequence if causal
//
// The two products and the softmax between them are those of the step kernel (step_tc.cu), and so is what bounds them: the exp unit at
// head_dim 64, the tensor core at 128 and 256. What is different is the work around them, which with short sequences is most of it.
//
// An item is a block of query tokens of one sequence and a KV head. A query tile of 128 rows holds the same tokens of `pack` query heads
// that share the KV head (one box of a 4-D tensor map), so that a tile has as few keys behind the diagonal as can be, and a sequence of 32
// tokens fills one where four heads share a KV head; a block takes two tiles of neighbouring tokens (head_dim 256: one). The items
// are numbered, those with the most key tiles first, and the blocks of one wave stay for the whole call and take one after the other:
// tensor memory, barriers and rings are set up once, and the next item's queries, keys and first scores come while the rows of the last
// one are written.
//
// Measured, us a launch in a CUDA graph, and the floor at the measured rate of a matrix product (1643 TFLOP/s):
//
//   16 prompts of up to 4099 rows, H32/kvH8 D128 bf16                   850 to 900   535
//   4 chunks of up to 1531 rows behind up to 16384, H32/kvH8 D128 bf16  655 to 695   483
//   2 documents of up to 32768 rows, H8 D64 fp16                        2060 to 2130 989 (1310 by the exp unit)
//   13 prompts of up to 200 rows, H24/kvH6 D64 bf16                     15 to 16     1.8
//   B1 H8 S8192, D32 / 64 / 128 / 256 bf16                              111 / 113 / 120 / 289
//
// The short ones are two items one after the other on some SMs, each a chain of copy, scores, softmax, product and way out of some 6 us.
// Items that blocks take over as they go replace a share dealt in advance, to and fro over the blocks: B1 H8 S32768 D64 1574 -> 1412 us, D128
// 2102 -> 1972.
//
// Roles (384 threads; head_dim 256 and one tile a block: 256): warp 0 copies with TMA, warps 1 and 2 issue tcgen05.mma (2: only where P has
// a place of its own, head_dim 64), warp 3 finds the items, warps 4 to 7 and 8 to 11 are the softmax of either tile, a row a thread.
//
// Two things that were slower: turns of the two softmax warps of a scheduler, by barriers (head_dim 64, 2 x 18944 rows: 247 -> 302 us); and other
// splits of the registers, which change the order of instructions more than the spills (72 / 216, 88 / 208, 104 / 200 of them at head_dim 64
// 247, 253, 230 us, at 128 281, 279, 283). Bytes spilled (stores / loads): head_dim 64 68 / 176, 128 72 / 76, 256 none; one tile a block, whose
// threads start with 128 registers, 108 / 260 and 272 / 392.
//
// Key tiles are counted from the sequence's first key. Of a query tile's last one only as many products are made as its rows see keys, in
// steps of 16, and only the halves of its scores that a warp's rows see are worked on; what a last step has of the next sequence is put
// out of V's tile before. A value of V that is not finite reaches queries of its own sequence whose weight for it is 0 where their query
// tile takes its key tile: 127 keys in front of it and 127 tokens in front of those at most.
#include <atomic>
#include <type_traits>

#include "mma16.cuh"
#include "tc_common.cuh"

namespace rab {

using namespace tcgen;

namespace {

struct PackedArgs {
  char* out;
  long long out_row, out_head;  // strides in elements
  float* lse;                   // (heads, rows) or NULL
  const int* ends;              // sequence b has query rows ends[b] to ends[b + 1]
  const int* k_ends;            // and keys
  int rows, k_rows, B, H, kvH, G;
  int pack, tile_tokens, tile_shift, token_shift;  // heads of a tile, its tokens and their log2, and log2 of a block's tokens
  int head_sets;                       // ceil(G / pack)
  int causal;
  int* status;
  unsigned long long wait_ns;
  int stall_after;
};

struct Item {
  int there;      // 0: the end
  int q0, q_len;  // first query row and rows of the sequence
  int k0, k_len;
  int token0;     // first token of the block
  int kv, head;   // KV head, first of the tile's heads inside the group
};

// kOne: one query tile a block and two blocks to an SM, for short sequences, of which a block's second tile would have few rows or none:
// two blocks are in different places of an item, so that one's copies and rows' way out run under the other's softmax.
template <int D, bool kOne>
struct PackedCfg {
  static_assert(!kOne || D <= 128, "two blocks to an SM");
  static constexpr int kTiles = D == 256 || kOne ? 1 : 2;
  static constexpr int kThreads = 128 + 128 * kTiles;
  static constexpr int kBN = D == 256 ? 64 : 128;  // keys of a tile
  static constexpr int kBoxes = D / 64;
  static constexpr int kQBytes = kBM * D * 2, kKvBytes = kBN * D * 2;
  static constexpr int kStages = (D == 64 ? 8 : 4) / (kOne ? 2 : 1);
  // head_dim 64: P has a place of its own and the next scores go out while P is made; 128: P overwrites S; 256: two score buffers, the
  // next but one scores go out behind the products with P that overwrites theirs
  static constexpr bool kEarlyS = D == 64, kDoubleS = D == 256, kOrdered = D == 128;
  static constexpr int kCols = kOne ? 256 : 512;  // of tensor memory
  static constexpr int kColS0 = 0, kColS1 = 128, kColO0 = kOne ? 128 : 256, kColO1 = 256 + D;
  static constexpr int kColP0 = !kEarlyS ? kColS0 : kOne ? 192 : 384, kColP1 = kEarlyS ? 448 : kColS1;
  // registers of the copying and issuing warps' threads and of the softmax threads: of 168 each at the start, or, two blocks to an SM, 128
  // (head_dim 256: 255 each, nothing to share out)
  static constexpr int kRegsLo = kOne ? 56 : D == 64 ? 104 : 72, kRegsHi = kOne ? 200 : D == 64 ? 200 : 216;
  static constexpr bool kShare = D != 256;
  static_assert(!kShare || 128 * kRegsLo + 128 * kTiles * kRegsHi <= kThreads * (kOne ? 128 : 168), "registers");
  static constexpr int kOffKv = kTiles * kQBytes;
  static constexpr int kOffOut = kOffKv + kStages * kKvBytes;  // rows on their way out: 4 KB a warp
  static constexpr int kOffBar = kOffOut + kTiles * 4 * 4096;
  static constexpr int kNumBars = 4 + 2 * kStages + 8 + 6;
  static constexpr int kOffNext = (kOffBar + kNumBars * 8 + 15) & ~15;  // the hardware's answer, see next_block
  static constexpr int kOffItem = kOffNext + 16;
  static constexpr int kSmemBytes = kOffItem + 2 * static_cast<int>(sizeof(Item)) + 16;
  static_assert((kOne ? 2 : 1) * (kSmemBytes + 1024) <= 228 * 1024, "shared memory");
};

// Key tiles that query tile w of an item needs (0: none, or no rows), and its keys.
__device__ inline int tile_keys(const PackedArgs& a, const Item& it, int w) {
  const int first = it.token0 + w * a.tile_tokens;
  if (first >= it.q_len) return 0;
  const int last = min(first + a.tile_tokens, it.q_len) - 1;
  return a.causal ? max(0, min(it.k_len, last + 1 + it.k_len - it.q_len)) : it.k_len;
}

// ---- items --------------------------------------------------------------------------

struct Seq {
  int q0, q_len, k0, k_len, blocks;
};
__device__ inline Seq sequence(const PackedArgs& a, int b) {
  Seq s;
  // (whatever the ends hold, no row outside the tensors is one of a sequence)
  s.q0 = min(max(a.ends[b], 0), a.rows);
  s.q_len = min(max(a.ends[b + 1], s.q0), a.rows) - s.q0;
  s.k0 = min(max(a.k_ends[b], 0), a.k_rows);
  s.k_len = min(max(a.k_ends[b + 1], s.k0), a.k_rows) - s.k0;
  s.blocks = static_cast<int>((static_cast<long long>(s.q_len) + (1 << a.token_shift) - 1) >> a.token_shift);
  return s;
}
// Blocks of a sequence that have c key tiles or more; they are its last ones.
template <int kBN>
__device__ inline int blocks_from(const PackedArgs& a, const Seq& s, int c) {
  if (c <= 0) return s.blocks;
  const long long behind = static_cast<long long>(c - 1) * kBN;  // more keys than these
  if (behind >= s.k_len) return 0;
  if (!a.causal) return s.blocks;
  const long long z = behind - s.k_len + s.q_len;
  const long long first = z < 0 ? 0 : z >> a.token_shift;
  return first >= s.blocks ? 0 : s.blocks - static_cast<int>(first);
}

// The items by their number, those with the most key tiles first, then by sequence, block, and KV head and set of heads. Run by a warp. What
// it has counted and where it has got to among the sequences it keeps, so that many sequences are gone over a few times for each number of
// key tiles and not for each item, nor for each number behind the last one (the grid has room for a block more of every sequence: of 32768
// places with one sequence of 300 rows among them, 8 KV heads, those were 886 a block, and other warps' waits ran out).
template <int kBN>
struct Items {
  const PackedArgs& a;
  int lane, of_block;  // items of a block of tokens
  Seq mine;            // lane's among the first 32 sequences
  int top, level;      // key tiles: the most, those of the last item found
  long long from, above;  // blocks with `level` key tiles or more, and with more than them
  long long all = -1;     // blocks, once they have been counted
  int chunk;              // sequences chunk to chunk + 31 have had `passed` blocks of just this level before them
  long long passed;
  __device__ Items(const PackedArgs& a_, int lane_) : a(a_), lane(lane_), of_block(a_.kvH * a_.head_sets) {
    mine = Seq{0, 0, 0, 0, 0};
    if (lane < a.B) mine = sequence(a, lane);
    int most = mine.k_len;
    for (int b = lane + 32; b < a.B; b += 32) most = max(most, sequence(a, b).k_len);
    most = __reduce_max_sync(0xffffffffu, most);
    top = (most + kBN - 1) / kBN;
    to_level(top);
  }
  __device__ Seq of(int b) const { return b < 32 ? mine : b < a.B ? sequence(a, b) : Seq{0, 0, 0, 0, 0}; }
  __device__ long long count(int c) const {  // blocks with c key tiles or more
    long long sum = __reduce_add_sync(0xffffffffu, blocks_from<kBN>(a, mine, c));
    for (int b0 = 32; b0 < a.B; b0 += 32) sum += __reduce_add_sync(0xffffffffu, blocks_from<kBN>(a, of(b0 + lane), c));
    return sum;
  }
  __device__ void to_level(int c) {
    level = c;
    from = count(c);
    above = count(c + 1);
    chunk = 0;
    passed = 0;
  }
  __device__ Item find(long long i) {
    Item it = {};
    const long long block = i / of_block;
    if (from <= block || above > block) {
      if (from <= block) {
        if (level == 0) return it;
        if (all < 0) all = count(0);
        if (all <= block) return it;
      }
      int lo = from <= block ? 0 : level + 1, hi = from <= block ? level : top + 1;  // count(lo) > block >= count(hi)
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (count(mid) > block) lo = mid;
        else hi = mid;
      }
      to_level(lo);
    }
    if (block - above < passed) chunk = 0, passed = 0;
    for (; chunk < a.B; chunk += 32) {
      const long long at = block - above - passed;  // among the blocks of just this level from here on
      const Seq s = of(chunk + lane);
      const int more = blocks_from<kBN>(a, s, level + 1), n = blocks_from<kBN>(a, s, level) - more;
      int upto = n;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
      }
      const unsigned has = __ballot_sync(0xffffffffu, upto > at);
      if (has) {
        const int src = __ffs(static_cast<int>(has)) - 1;
        const int m = static_cast<int>(i - block * of_block);
        it.there = 1;
        it.q0 = __shfl_sync(0xffffffffu, s.q0, src);
        it.q_len = __shfl_sync(0xffffffffu, s.q_len, src);
        it.k0 = __shfl_sync(0xffffffffu, s.k0, src);
        it.k_len = __shfl_sync(0xffffffffu, s.k_len, src);
        const int nth = static_cast<int>(at) - __shfl_sync(0xffffffffu, upto - n, src);
        it.token0 = (__shfl_sync(0xffffffffu, s.blocks - more, src) - 1 - nth) << a.token_shift;
        it.kv = m % a.kvH;
        it.head = m / a.kvH * a.pack;
        return it;
      }
      passed += __shfl_sync(0xffffffffu, upto, 31);
    }
    return it;
  }
};

__device__ inline void tma_load_4d(unsigned dst, const CUtensorMap* map, unsigned bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// Takes the next block of the grid that has not begun in its place: *number is its number; *more: there was one (if not, no further one
// may be asked for). The answer goes to 16 bytes at `room` and `bar`; n counts the calls. Run by a warp; false: the wait ran out.
template <typename Wait>
__device__ inline bool take_block(unsigned room, unsigned bar, int n, unsigned* number, bool* more, Wait wait) {
  if ((threadIdx.x & 31) == 0) {
    mbar_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(room), "r"(bar)
                 : "memory");
  }
  __syncwarp();
  if (!wait(bar, n & 1, 14, n)) return false;
  unsigned got, x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 answer;\n\t"
      "ld.shared.b128 answer, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, answer;\n\t"
      "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, answer;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(room)
      : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (the next answer comes behind this reading)
  __syncwarp();
  *more = got != 0;
  *number = x;
  return true;
}

// ---- kernel -------------------------------------------------------------------------

// DR: head_dim of the tensors: D, or 32 on the 64-wide kernel, whose copies bring zeros for the upper half of every row.
template <int D, int DR, typename T, bool kOne>
__global__ void __launch_bounds__(PackedCfg<D, kOne>::kThreads, kOne ? 2 : 1)
    packed_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PackedArgs a) {
  using C = PackedCfg<D, kOne>;
  constexpr int kBN = C::kBN;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) unsigned char smem[];
  const unsigned base = smem_u32(smem), s_kv = base + C::kOffKv, bars = base + C::kOffBar;
  const unsigned q_full = bars, q_free = bars + 16;                                      // [2] each
  const unsigned kv_full = bars + 32, kv_free = kv_full + 8 * C::kStages;                // [kStages]
  const unsigned s_full = kv_free + 8 * C::kStages, s_free = s_full + 16;                // [2]
  const unsigned p_full = s_free + 16, o_done = p_full + 16;                             // [2]
  const unsigned item_full = o_done + 16, item_free = item_full + 16;                    // [2]
  const unsigned next_full = item_free + 16, copied = next_full + 8;
  volatile Item* const items = reinterpret_cast<volatile Item*>(smem + C::kOffItem);
  unsigned* const tmem_slot = reinterpret_cast<unsigned*>(smem + C::kOffItem + 2 * sizeof(Item));
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int kIssuers = C::kEarlyS ? C::kTiles : 1, kItemReaders = 1 + kIssuers + 4 * C::kTiles;
  let_next_start();
  if (tid == 0) {
    for (int w = 0; w < 2; ++w) {
      mbar_init(q_full + 8 * w, 1);
      mbar_init(q_free + 8 * w, 1);
      mbar_init(s_full + 8 * w, 1);
      mbar_init(s_free + 8 * w, kBM);
      mbar_init(p_full + 8 * w, kBM);
      mbar_init(o_done + 8 * w, 1);
      mbar_init(item_full + 8 * w, 1);
      mbar_init(item_free + 8 * w, kItemReaders);
    }
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(kv_full + 8 * s, 1);
      mbar_init(kv_free + 8 * s, kIssuers);
    }
    mbar_init(next_full, 1);
    mbar_init(copied, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&map_q);
    prefetch_map(&map_k);
    prefetch_map(&map_v);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(C::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = *tmem_slot;
  wait_for_previous();
  // a launch before this one gave up: nothing is computed until the word is read
  const bool gone = __syncthreads_or(tid == 0 && *reinterpret_cast<volatile int*>(a.status) != 0) != 0;

  auto wait = [&](unsigned bar, unsigned parity, int which, int n) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.status, which, n, a.wait_ns)) != 0;
  };
  // The n-th item of this block; false: there is none, or the block gives up.
  auto item_at = [&](int n) {
    const volatile Item& from = items[n & 1];
    Item it;
    it.there = from.there, it.q0 = from.q0, it.q_len = from.q_len, it.k0 = from.k0, it.k_len = from.k_len;
    it.token0 = from.token0, it.kv = from.kv, it.head = from.head;
    return it;
  };
  auto give_item_back = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(item_free + 8 * (n & 1));
  };
  auto next_item = [&](int n, Item* it) {
    if (!wait(item_full + 8 * (n & 1), (n >> 1) & 1, 11, n)) return false;
    *it = item_at(n);
    give_item_back(n);
    return it->there != 0;
  };
  auto tiles_of = [&](const Item& it, int w) { return w < C::kTiles ? (tile_keys(a, it, w) + kBN - 1) / kBN : 0; };

  if (warp < 4) {
    if constexpr (C::kShare) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsLo));
    if (gone) {
    } else if (warp == 3) {
      // ------------------------------------------------------------------ items ----
      // The grid has a block for every item that there can be, of which one for each SM runs. Its first item is that of its own number;
      // then it takes over the numbers of blocks that have not begun, in the order in which they would, as long as there are any.
      Items<kBN> list(a, lane);
      bool ok = true, more = true;
      int taken = 0;
      unsigned number = blockIdx.x;
      for (int n = 0; ok; ++n) {
        Item it = {};
        if (more) it = list.find(number);
        // (the rest of the grid has nothing to do: it is taken over as well, so that it does not have to begin)
        while (more && !it.there && ok) {
          ok = take_block(base + C::kOffNext, next_full, taken++, &number, &more, wait);
          if (ok && more) it = list.find(number);
        }
        if (!ok) break;
        if (n >= 2) ok = wait(item_free + 8 * (n & 1), ((n >> 1) + 1) & 1, 12, n);
        if (!ok) break;
        if (lane == 0) {
          volatile Item& to = items[n & 1];
          to.there = it.there, to.q0 = it.q0, to.q_len = it.q_len, to.k0 = it.k0, to.k_len = it.k_len;
          to.token0 = it.token0, to.kv = it.kv, to.head = it.head;
          mbar_arrive(item_full + 8 * (n & 1));
        }
        __syncwarp();
        if (!it.there) break;
        // not before the item's last copy is on its way: what is taken early is another block's late
        ok = wait(copied, n & 1, 15, n) && take_block(base + C::kOffNext, next_full, taken++, &number, &more, wait);
      }
    } else if (warp == 0) {
      // ----------------------------------------------------------------- copies ----
      unsigned ring = 0, q_uses[2] = {0, 0};
      bool ok = true;
      Item it;
      for (int n = 0; ok && next_item(n, &it); ++n) {
        const int n_of[2] = {tiles_of(it, 0), tiles_of(it, 1)}, n_tiles = max(n_of[0], n_of[1]);
        for (int w = 0; w < C::kTiles && ok; ++w) {
          if (n_of[w] == 0) continue;
          if (q_uses[w] > 0) ok = wait(q_free + 8 * w, (q_uses[w] + 1) & 1, 13, n);
          ++q_uses[w];
          if (ok && lane == 0) {
            mbar_expect_tx(q_full + 8 * w, C::kQBytes);
            for (int bx = 0; bx < C::kBoxes; ++bx)
              tma_load_4d(base + w * C::kQBytes + bx * (kBM * 128), &map_q, q_full + 8 * w, bx * 64,
                          it.q0 + it.token0 + w * a.tile_tokens, it.kv, it.head);
          }
        }
        for (int t = 0; t < n_tiles && ok; ++t)
          for (int which = 0; which < 2 && ok; ++which, ++ring) {
            const unsigned slot = ring % C::kStages, use = ring / C::kStages;
            if (use > 0) ok = wait(kv_free + 8 * slot, (use + 1) & 1, 1, ring);
            if (a.stall_after >= 0 && static_cast<int>(ring) >= a.stall_after) ok = false;  // (test hook)
            if (ok && lane == 0) {
              mbar_expect_tx(kv_full + 8 * slot, C::kKvBytes);
              for (int bx = 0; bx < C::kBoxes; ++bx)
                tma_load_3d(s_kv + slot * C::kKvBytes + bx * (kBN * 128), which == 0 ? &map_k : &map_v, kv_full + 8 * slot, bx * 64,
                            it.k0 + t * kBN, it.kv);
            }
          }
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(copied);
      }
    } else if (warp <= kIssuers) {
      // --------------------------------------------------------------- products ----
      constexpr unsigned kFmt = kBf16 ? 1u : 0u;
      constexpr unsigned idesc_pv = make_idesc(kFmt, 1, D, kBM);
      constexpr unsigned kBox = (kBM * 128) >> 4, kKvBox = (kBN * 128) >> 4;
      const unsigned long long qd0 = desc_kmajor(base), kd0 = desc_kmajor(s_kv), vd0 = desc_mnmajor(s_kv, kBN * 128, 1024);
      unsigned ring = 0;  // key tiles of this block so far, twice
      auto slot_of = [&](unsigned i) { return i % C::kStages; };
      auto wait_kv = [&](unsigned i) { return wait(kv_full + 8 * slot_of(i), (i / C::kStages) & 1, 4, i); };
      auto put_s = [&](unsigned i, unsigned col, int w, int steps) {  // S = Q_w K^T of ring item i, of `steps` times 16 keys
        const unsigned idesc_s = make_idesc(kFmt, 0, 16, kBM) + (static_cast<unsigned>(steps - 1) << 18);
        const unsigned long long qd = qd0 + static_cast<unsigned long long>(w * (C::kQBytes >> 4));
        const unsigned long long kd = kd0 + static_cast<unsigned long long>(slot_of(i) * (C::kKvBytes >> 4));
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          mma_ss(tmem + col, qd + (ks / 4) * kBox + (ks % 4) * 2, kd + (ks / 4) * kKvBox + (ks % 4) * 2, idesc_s, ks > 0);
      };
      auto put_pv = [&](unsigned i, unsigned col_o, unsigned col_p, int steps, bool acc) {  // O += P V, `steps` times 16 keys
        const unsigned long long vd = vd0 + static_cast<unsigned long long>(slot_of(i) * (C::kKvBytes >> 4));
        if (steps == kBN / 16) {
#pragma unroll
          for (int ks = 0; ks < kBN / 16; ++ks) mma_ts(tmem + col_o, tmem + col_p + ks * 8, vd + ks * (2048 >> 4), idesc_pv, acc || ks > 0);
        } else {
          for (int ks = 0; ks < steps; ++ks) mma_ts(tmem + col_o, tmem + col_p + ks * 8, vd + ks * (2048 >> 4), idesc_pv, acc || ks > 0);
        }
      };
      // V's rows behind the sequence's last key, as far as the last step of 16 reaches (its weights there are 0, but 0 times what another
      // sequence has there need not be). Both issuing warps may do it: they write the same zeros.
      auto clear_v = [&](unsigned i, int keys) {
        if (keys >= kBN || keys % 16 == 0) return;
        const unsigned tile = s_kv + slot_of(i) * C::kKvBytes + keys * 128;
        for (int x = lane; x < (16 - keys % 16) * 8 * C::kBoxes; x += 32)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + x / 8 % (16 - keys % 16) * 128 + x / (8 * (16 - keys % 16)) * (kBN * 128) + x % 8 * 16),
                       "r"(0)
                       : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      };
      bool ok = true;
      Item it;
      int q_uses[2] = {0, 0}, p_uses[2] = {0, 0}, s_uses = 0;
      for (int n = 0; ok && next_item(n, &it); ++n) {
        const int n_of[2] = {tiles_of(it, 0), tiles_of(it, 1)}, n_tiles = max(n_of[0], n_of[1]);
        auto keys_of = [&](int t) { return it.k_len - t * kBN; };  // of the sequence, from a tile on
        const int seen_of[2] = {tile_keys(a, it, 0), C::kTiles == 2 ? tile_keys(a, it, 1) : 0};
        // keys of tile t that some row of query tile w sees, in steps of 16
        auto steps_of = [&](int t, int w) { return min(kBN, (seen_of[w] - t * kBN + 15) & ~15) / 16; };
        if constexpr (C::kOrdered) {
          // One warp issues for both tiles in turn: P.V of tile t and, behind it, the scores of tile t + 1 over the P that it read.
          ok = n_tiles == 0 || wait_kv(ring);
          for (int w = 0; w < 2 && ok; ++w) {
            if (n_of[w] == 0) continue;
            ok = wait(q_full + 8 * w, q_uses[w]++ & 1, 3, n);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              put_s(ring, w == 0 ? C::kColS0 : C::kColS1, w, steps_of(0, w));
              tc_commit(s_full + 8 * w);
              if (n_of[w] == 1) tc_commit(q_free + 8 * w);
              if (w == 1 || n_of[1] == 0) tc_commit(kv_free + 8 * slot_of(ring));
            }
            __syncwarp();
          }
          for (int t = 0; t < n_tiles && ok; ++t) {
            const unsigned iv = ring + 2 * t + 1, ik = iv + 1;
            ok = wait_kv(iv) && (t + 1 >= n_tiles || wait_kv(ik));
            if (!ok) break;
            clear_v(iv, keys_of(t));
            for (int w = 0; w < 2 && ok; ++w) {
              if (t >= n_of[w]) continue;
              ok = wait(p_full + 8 * w, p_uses[w]++ & 1, 6, t);
              if (!ok) break;
              tc_fence_after();
              if (elect_one()) {
                put_pv(iv, w == 0 ? C::kColO0 : C::kColO1, w == 0 ? C::kColP0 : C::kColP1, steps_of(t, w), t > 0);
                const bool last_v = w == 1 || t >= n_of[1];
                if (t + 1 < n_of[w]) {
                  put_s(ik, w == 0 ? C::kColS0 : C::kColS1, w, steps_of(t + 1, w));
                  tc_commit(s_full + 8 * w);
                  if (t + 2 == n_of[w]) tc_commit(q_free + 8 * w);
                } else {
                  tc_commit(o_done + 8 * w);
                }
                if (last_v) {
                  tc_commit(kv_free + 8 * slot_of(iv));
                  if (t + 1 < n_tiles) tc_commit(kv_free + 8 * slot_of(ik));
                }
              }
              __syncwarp();
            }
          }
        } else if constexpr (C::kDoubleS) {
          auto do_s = [&](int t) {
            if (!wait_kv(ring + 2 * t)) return false;
            tc_fence_after();
            if (elect_one()) {
              const int buf = s_uses & 1;
              put_s(ring + 2 * t, buf * kBN, 0, steps_of(t, 0));
              tc_commit(s_full + 8 * buf);
              tc_commit(kv_free + 8 * slot_of(ring + 2 * t));
              if (t + 1 == n_tiles) tc_commit(q_free);
            }
            __syncwarp();
            ++s_uses;
            return true;
          };
          if (n_tiles > 0) ok = wait(q_full, q_uses[0]++ & 1, 3, n) && do_s(0);
          if (n_tiles > 1) ok = ok && do_s(1);
          for (int t = 0; t < n_tiles && ok; ++t) {
            ok = wait(p_full, p_uses[0] & 1, 6, t) && wait_kv(ring + 2 * t + 1);
            if (!ok) break;
            clear_v(ring + 2 * t + 1, keys_of(t));
            tc_fence_after();
            if (elect_one()) {
              put_pv(ring + 2 * t + 1, C::kColO0, (p_uses[0] & 1) * kBN, steps_of(t, 0), t > 0);
              tc_commit(o_done);
              tc_commit(kv_free + 8 * slot_of(ring + 2 * t + 1));
            }
            __syncwarp();
            ++p_uses[0];
            if (t + 2 < n_tiles) ok = do_s(t + 2);
          }
        } else {
          // A warp to a tile: S(t + 1) as soon as the softmax threads hold S(t), P.V of tile t when its P is written.
          const int w = warp - 1, mine = n_of[w];
          const unsigned col_s = w == 0 ? C::kColS0 : C::kColS1;
          auto do_s = [&](int t) {
            const unsigned i = ring + 2 * t;
            if (!wait_kv(i)) return false;
            tc_fence_after();
            if (elect_one()) {
              put_s(i, col_s, w, steps_of(t, w));
              tc_commit(s_full + 8 * w);
              tc_commit(kv_free + 8 * slot_of(i));
              if (t + 1 == mine) tc_commit(q_free + 8 * w);
            }
            __syncwarp();
            return true;
          };
          auto give_back = [&](unsigned i) {  // a tile of the other query tile alone: its place goes back unread
            if (!wait_kv(i)) return false;
            if (lane == 0) mbar_arrive(kv_free + 8 * slot_of(i));
            __syncwarp();
            return true;
          };
          if (mine > 0) ok = wait(q_full + 8 * w, q_uses[0]++ & 1, 3, n) && do_s(0);
          for (int t = 0; t < n_tiles && ok; ++t) {
            const unsigned iv = ring + 2 * t + 1;
            if (t < mine) {
              if (t + 1 < mine) ok = wait(s_free + 8 * w, p_uses[0] & 1, 9, t) && do_s(t + 1);
              ok = ok && wait(p_full + 8 * w, p_uses[0] & 1, 6, t) && wait_kv(iv);
              if (!ok) break;
              ++p_uses[0];
              clear_v(iv, keys_of(t));
              tc_fence_after();
              if (elect_one()) {
                put_pv(iv, w == 0 ? C::kColO0 : C::kColO1, w == 0 ? C::kColP0 : C::kColP1, steps_of(t, w), t > 0);
                tc_commit(o_done + 8 * w);
                tc_commit(kv_free + 8 * slot_of(iv));
              }
              __syncwarp();
            } else {
              ok = give_back(ring + 2 * t) && give_back(iv);
            }
          }
        }
        ring += 2 * n_tiles;
      }
    }
  } else {
    if constexpr (C::kShare) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsHi));
    // ----------------------------------------------------------------- softmax ----
    const int w = (warp - 4) >> 2;
    const int row = ((warp & 3) << 5) + lane;
    const unsigned lane_base = static_cast<unsigned>((warp & 3) << 5) << 16;
    const unsigned t_s = tmem + lane_base + (w == 0 ? C::kColS0 : C::kColS1);
    const unsigned t_o = tmem + lane_base + (w == 0 ? C::kColO0 : C::kColO1);
    const unsigned t_p = tmem + lane_base + (w == 0 ? C::kColP0 : C::kColP1);
    const unsigned stage = base + C::kOffOut + (warp - 4) * 4096;
    const float scale_log2 = rsqrtf(static_cast<float>(DR)) * kLog2e;
    bool ok = !gone;
    unsigned uses = 0, items_of = 0;  // key tiles and items of this query tile so far
    // (what the rows' way out wants of the item is read again behind the tile loop, which has no registers for it)
    auto place = [&](const Item& it, int* head, int* token) {
      *head = it.head + (row >> a.tile_shift);
      *token = it.token0 + (w << a.tile_shift) + (row & (a.tile_tokens - 1));
      return *token < it.q_len && *head < a.G;
    };
    for (int n = 0; ok; ++n) {
      ok = wait(item_full + 8 * (n & 1), (n >> 1) & 1, 11, n);
      if (!ok) break;
      int n_own, see;
      bool valid;
      {
        const Item it = item_at(n);
        if (!it.there) break;
        int head, token;
        valid = place(it, &head, &token);
        n_own = tiles_of(it, w);
        // keys that the row sees (a row that there is not: all, with weights of 0, so that it asks for no mask)
        see = !valid ? 0x7fffffff : a.causal ? min(it.k_len, token + 1 + it.k_len - it.q_len) : it.k_len;
      }
      const bool any_valid = __any_sync(0xffffffffu, valid) != 0;
      float m_ref = valid ? -INFINITY : 1e30f, l_run = 0.f;
      for (int j = 0; j < n_own && ok; ++j, ++uses) {
        const int buf = C::kDoubleS ? uses & 1 : 0;
        ok = wait(s_full + 8 * (C::kDoubleS ? buf : w), C::kDoubleS ? (uses >> 1) & 1 : uses & 1, 7, j);
        if (!ok) break;
        tc_fence_after();
        // The P that is about to be overwritten has been read where P has a place of its own (P.V(j - 1), issued a softmax ago) or, with
        // two buffers, once O is to be rescaled.
        auto wait_pv = [&]() {
          if constexpr (!C::kOrdered) {
            if (j > 0) {
              ok = wait(o_done + 8 * w, (uses - 1) & 1, 10, j);
              if (ok) tc_fence_after();
            }
          }
        };
        if (!any_valid) {
          if constexpr (C::kEarlyS) mbar_arrive(s_free + 8 * w);
          wait_pv();
          if (!ok) break;
          mbar_arrive(p_full + 8 * w);
          continue;
        }
        const int hi = min(max(see - j * kBN, 0), kBN);  // columns that the row sees
        const bool full = __all_sync(0xffffffffu, hi == kBN) != 0;
        // The first kCols columns of the tile (64 of 128 where no row of the warp sees more: the others' weights are 0); false: gave up.
        auto work = [&](auto cols) {
          constexpr int kCols = decltype(cols)::value;
          float s[kCols];
          if constexpr (kCols == 128) tmem_ld128(t_s, s);
          else tmem_ld64(t_s + buf * kBN, s);
          if constexpr (C::kEarlyS) {
            tc_fence_before();
            mbar_arrive(s_free + 8 * w);
          }
          if (!full) {
#pragma unroll
            for (int i = 0; i < kCols; ++i) s[i] = i < hi ? s[i] : -INFINITY;
          }
          // P = 2^(s scale - m_ref) and the row sum; m_ref is moved only when a tile's sum says so (see step_tc.cu)
          const float2 scale2 = make_float2(scale_log2, scale_log2);
          float2 sum_a, sum_b;
          auto half_tile = [&](int h, float neg_m) {
            const float2 negm2 = make_float2(neg_m, neg_m);
            unsigned pk[32];
#pragma unroll
            for (int i = 0; i < 64; i += 4) {
              const int c = h * 64 + i;
              const float2 x0 = ffma2(make_float2(s[c], s[c + 1]), scale2, negm2);
              const float2 x1 = ffma2(make_float2(s[c + 2], s[c + 3]), scale2, negm2);
              const float2 p0 = make_float2(ex2(x0.x), ex2(x0.y)), p1 = make_float2(ex2(x1.x), ex2(x1.y));
              sum_a = fadd2(sum_a, p0);
              sum_b = fadd2(sum_b, p1);
              pk[i / 2] = pack_pair<T>(p0.x, p0.y);
              pk[i / 2 + 1] = pack_pair<T>(p1.x, p1.y);
            }
            tmem_st32u(t_p + buf * kBN + h * 32, &pk[0]);
          };
          auto whole_tile = [&]() {
            const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
            sum_a = sum_b = make_float2(0.f, 0.f);
#pragma unroll
            for (int h = 0; h < kCols / 64; ++h) half_tile(h, neg_m);
            if constexpr (kCols < kBN) {
              unsigned none[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) none[i] = 0u;
              tmem_st32u(t_p + 32, &none[0]);
            }
            return (sum_a.x + sum_a.y) + (sum_b.x + sum_b.y);
          };
          bool need = m_ref == -INFINITY && hi > 0;  // this row's reference has to move
          bool slow = __any_sync(0xffffffffu, need) != 0;
          float row_sum = 0.f;
          [[maybe_unused]] bool waited = slow;
          if (C::kEarlyS || slow) wait_pv();
          if (!ok) return;
          if (!slow) {
            row_sum = whole_tile();
            need = !(row_sum <= kRowSumLimit) && valid;  // (NaN too)
            slow = __any_sync(0xffffffffu, need) != 0;
            if (C::kDoubleS && slow) wait_pv(), waited = true;  // O has to be at rest
            if (!ok) return;
          }
          // Rows that need it move their reference, the others keep theirs, so that no row's result hangs on which rows share its warp.
          // Those that have one and were not asked yet, because another's first tile is here, may need it in turn.
#pragma unroll 1
          for (int pass = 0; slow && pass < 2; ++pass) {
            float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
            for (int i = 4; i < kCols; i += 8) {
              m0 = max3(m0, s[i], s[i + 1]);
              m1 = max3(m1, s[i + 2], s[i + 3]);
              if (i + 4 < kCols) {
                m2 = max3(m2, s[i + 4], s[i + 5]);
                m3 = max3(m3, s[i + 6], s[i + 7]);
              }
            }
            const float tile_max = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * scale_log2;
            float alpha = 1.f;
            bool rescale = false;
            if (need && tile_max > m_ref) {
              if (m_ref > -INFINITY) {
                alpha = ex2(m_ref - tile_max);
                rescale = true;
              }
              m_ref = tile_max;
            }
            if (j > 0 && __any_sync(0xffffffffu, rescale)) {
              l_run *= alpha;
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                float o[32];
                tmem_ld32(t_o + c * 32, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= alpha;
                tmem_st32(t_o + c * 32, o);
              }
            }
            row_sum = whole_tile();
            need = !(row_sum <= kRowSumLimit) && valid;
            slow = __any_sync(0xffffffffu, need) != 0;
          }
          l_run += row_sum;
          if constexpr (C::kDoubleS) {  // (keeps step with the barrier, which tells the latest phase from the one before alone)
            if (!waited) wait_pv();
          }
        };
        if constexpr (kBN == 128) {
          if (!full && !__any_sync(0xffffffffu, valid && hi > 64)) work(std::integral_constant<int, 64>());
          else work(std::integral_constant<int, 128>());
        } else {
          work(std::integral_constant<int, 64>());
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_full + 8 * w);
      }
      if (!ok) break;
      // ---------------------------------------------------------------- epilogue ----
      if (n_own > 0) {
        ok = wait(o_done + 8 * w, (C::kOrdered ? items_of : uses - 1) & 1, 8, n);
        if (!ok) break;
        tc_fence_after();
        ++items_of;
      }
      const Item it = item_at(n);
      give_item_back(n);
      if (!any_valid) continue;
      int head, token;
      place(it, &head, &token);
      // (scores of NaN alone set no reference, but the row is NaN and not one without keys)
      const bool have = n_own > 0 && (m_ref > -INFINITY || l_run != l_run);
      const float inv = have ? 1.f / l_run : 0.f;
      if (a.lse && valid)
        a.lse[static_cast<size_t>(head * a.kvH + it.kv) * a.rows + it.q0 + token] = !have ? -INFINITY : l_run > 0.f ? m_ref * kLn2 + logf(l_run) : l_run;
      const unsigned rows_there = __ballot_sync(0xffffffffu, valid);
      // 64 columns at a time through shared memory, so that 8 lanes write 128 bytes of a row side by side
      constexpr int kCols = DR < 64 ? DR : 64, kLanes = kCols / 8, kRowsPer = 32 / kLanes;
      // (the lane out of its register, volatile: what hangs on threadIdx the compiler works out in front of the tile loop, and carries
      // through it in registers that the loop lacks)
      int lane_out;
      asm volatile("mov.u32 %0, %%laneid;" : "=r"(lane_out));
      const int piece = lane_out % kLanes, first = lane_out / kLanes;
#pragma unroll 1
      for (int pass = 0; pass < DR / kCols; ++pass) {
        float o[64];
        if (n_own > 0) {
          if constexpr (kCols == 64) tmem_ld64(t_o + pass * kCols, o);
          else tmem_ld32(t_o, reinterpret_cast<float(&)[32]>(o));
        } else {
#pragma unroll
          for (int i = 0; i < kCols; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < kCols; ++i) o[i] = have ? o[i] * inv : 0.f;
#pragma unroll
        for (int i = 0; i < kCols / 8; ++i)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane_out * 128 + ((i ^ (lane_out & 7)) << 4)),
                       "r"(pack_pair<T>(o[8 * i], o[8 * i + 1])), "r"(pack_pair<T>(o[8 * i + 2], o[8 * i + 3])),
                       "r"(pack_pair<T>(o[8 * i + 4], o[8 * i + 5])), "r"(pack_pair<T>(o[8 * i + 6], o[8 * i + 7]))
                       : "memory");
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 32 / kRowsPer; ++i) {
          const int r = i * kRowsPer + first, of_tile = ((warp & 3) << 5) + r;
          const int h = (it.head + (of_tile >> a.tile_shift)) * a.kvH + it.kv;
          const int q = it.q0 + it.token0 + (w << a.tile_shift) + (of_tile & (a.tile_tokens - 1));
          uint4 v;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(stage + r * 128 + ((piece ^ (r & 7)) << 4)));
          if (rows_there >> r & 1u)
            *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + q * a.out_row + h * a.out_head + pass * kCols + piece * 8) = v;
        }
        __syncwarp();
      }
      tc_fence_before();  // (the next item's products write O once this thread has brought its P)
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (*abort_flag) {  // give copies and products in flight time to land
      const unsigned long long t0 = global_ns();
      while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::kCols) : "memory");
  }
}

// ---- host side ----------------------------------------------------------------------

// 16-bit rows as a tensor map of `rank` dimensions of `dims` elements, strides in elements, boxes of 64 columns, 128B swizzle.
int make_rows_map(CUtensorMap* map, bool bf16, const void* base, int rank, const cuuint64_t* dims, const long long* strides,
                  const cuuint32_t* box) {
  EncodeTiledFn fn = encode_fn();
  RAB_REQUIRE(fn != nullptr, RA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t bytes[4];
  for (int i = 0; i + 1 < rank; ++i) bytes[i] = static_cast<cuuint64_t>(strides[i]) * 2;
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base), dims,
                        bytes, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RAB_REQUIRE(r == CUDA_SUCCESS, RA_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", static_cast<int>(r));
  return RA_OK;
}

// Heads of a query tile: the power of two that makes the fewest tiles, the largest of those that are alike.
int heads_per_tile(int G, long long tokens) {
  int best = 1;
  long long least = -1;
  for (int p = 1; p <= 16 && p < 2 * G; p *= 2) {
    const long long per = kBM / p, tiles = (G + p - 1) / p * ((tokens + per - 1) / per);
    if (least < 0 || tiles <= least) least = tiles, best = p;
  }
  return best;
}

// Rows that TMA can copy: 16-byte aligned, and strides of a row or more.
bool rows_for_tma(const ra_rows& r, int head_dim, int heads, int rows) {
  unsigned long long all = reinterpret_cast<uintptr_t>(r.data);
  if (heads > 1) all |= static_cast<unsigned long long>(r.head_stride) * 2;
  if (rows > 1) all |= static_cast<unsigned long long>(r.row_stride) * 2;
  return (all & 15u) == 0 && (heads <= 1 || r.head_stride >= head_dim) && (rows <= 1 || r.row_stride >= head_dim) &&
         (heads <= 1 || r.head_stride < 1ll << 32) && (rows <= 1 || r.row_stride < 1ll << 32);
}

template <int D, int DR, typename T, bool kOne>
int launch_tiles(const ra_rows& q, const ra_rows& k, const ra_rows& v, PackedArgs a, cudaStream_t stream) {
  using C = PackedCfg<D, kOne>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  a.token_shift = 0;
  while ((1 << a.token_shift) < C::kTiles * a.tile_tokens) ++a.token_shift;
  CUtensorMap mq, mk, mv;
  auto step = [&](long long stride, int n) { return n > 1 ? stride : static_cast<long long>(DR); };  // (of one row or head: any)
  const long long qh = step(q.head_stride, a.H);
  const cuuint64_t qdims[4] = {DR, static_cast<cuuint64_t>(a.rows), static_cast<cuuint64_t>(a.kvH), static_cast<cuuint64_t>(a.G)};
  const long long qstrides[3] = {step(q.row_stride, a.rows), qh, qh * a.kvH};
  const cuuint32_t qbox[4] = {64, static_cast<cuuint32_t>(a.tile_tokens), 1, static_cast<cuuint32_t>(a.pack)};
  int rc = make_rows_map(&mq, kBf16, q.data, 4, qdims, qstrides, qbox);
  if (rc != RA_OK) return rc;
  const cuuint64_t kdims[3] = {DR, static_cast<cuuint64_t>(std::max(a.k_rows, 1)), static_cast<cuuint64_t>(a.kvH)};
  const cuuint32_t kbox[3] = {64, C::kBN, 1};
  const long long ks[2] = {step(k.row_stride, a.k_rows), step(k.head_stride, a.kvH)}, vs[2] = {step(v.row_stride, a.k_rows), step(v.head_stride, a.kvH)};
  rc = make_rows_map(&mk, kBf16, k.data, 3, kdims, ks, kbox);
  if (rc == RA_OK) rc = make_rows_map(&mv, kBf16, v.data, 3, kdims, vs, kbox);
  if (rc != RA_OK) return rc;
  auto kern = packed_kernel<D, DR, T, kOne>;
  static std::atomic<unsigned long long> smem_set{0};  // once per device and instantiation
  int dev = 0;
  RAB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !(smem_set.load(std::memory_order_acquire) >> dev & 1ull)) {
    RAB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    if (dev >= 0 && dev < 64) smem_set.fetch_or(1ull << dev, std::memory_order_release);
  }
  // (as many items as there can be)
  const long long most = ((static_cast<long long>(a.rows) >> a.token_shift) + a.B) * a.kvH * a.head_sets;
  RAB_REQUIRE(most < 1ll << 31, RA_ERR_INVALID, "packed_attention: too many rows, sequences and heads");
  RAB_CUDA(launch_overlapped(kern, dim3(static_cast<unsigned>(most)), dim3(C::kThreads), C::kSmemBytes, stream, mq, mk, mv, a));
  return RA_OK;
}

template <int D, int DR, typename T>
int launch_packed(const ra_rows& q, const ra_rows& k, const ra_rows& v, PackedArgs a, cudaStream_t stream) {
  const long long tokens = (a.rows + a.B - 1) / a.B;
  a.pack = heads_per_tile(a.G, tokens);
  a.tile_tokens = kBM / a.pack;
  while ((1 << a.tile_shift) < a.tile_tokens) ++a.tile_shift;
  a.head_sets = (a.G + a.pack - 1) / a.pack;
  if constexpr (D <= 128) {
    // Sequences of one query tile on average, and at head_dim 64 and below of two if their keys are few, are taken a tile a block. us in a
    // graph, a tile a block / two:
    //   16384 rows, H32/kvH8 D128 (a tile is 32 tokens), sequences of 16, 32, 64, 128 rows: 162 / 252, 91 / 127, 87 / 81, 102 / 87
    //   16384 rows, H24/kvH6 D64 (32 tokens), sequences of 32, 64, 128 rows: 57 / 101, 54 / 55, 62 / 61
    //   16384 rows, H16 D64 (128 tokens), sequences of 128, 256, 512 rows: 49 / 85, 56 / 67, 69 / 75
    //   64 chunks on 8192 keys, 32 rows of H32/kvH8 D128: 416 / 552, 64 rows of H24/kvH6 D64: 366 / 328
    // A call of few sequences, where all items run at once, feels it little: 5 to 40 prompts of up to 50 to 200 rows 0.85 to 1.11.
    // The host knows rows and places but no lengths: a place without a sequence counts as a short one, room without rows as rows. One
    // prompt of 8192 rows in 1, 16, 256 places (H32/kvH8 D128), as chosen: 432, 482, 625 us, the last 525 with two tiles a block; a fixed
    // number of places well above the sequences of most steps, or a long prompt among hundreds of short ones, pays for it here and in the
    // finder of items, which goes over all places for every number of key tiles.
    constexpr int kFewKeys = 512;
    const bool two = D == 64 && a.k_rows <= static_cast<long long>(kFewKeys) * a.B;
    if (tokens <= (two ? 2 : 1) * a.tile_tokens) return launch_tiles<D, DR, T, true>(q, k, v, a, stream);
  }
  return launch_tiles<D, DR, T, false>(q, k, v, a, stream);
}

}  // namespace
}  // namespace rab

using namespace rab;

extern "C" int ra_packed_attention(int dtype, const ra_rows* q, const ra_rows* k, const ra_rows* v, const ra_rows* out, float* lse,
                                   const ra_shape* shape, const int* ends, const int* k_ends, int causal, ra_stream stream_) {
  const char* const what = "packed_attention";
  RAB_REQUIRE(q && k && v && out && shape, RA_ERR_INVALID, "%s: null argument", what);
  RAB_REQUIRE(dtype == RA_F16 || dtype == RA_BF16, RA_ERR_INVALID, "%s: rows are fp16 or bf16, got dtype %d", what, dtype);
  const int D = shape->head_dim, H = shape->heads, kvH = kv_heads_of(*shape);
  RAB_REQUIRE(D == 32 || D == 64 || D == 128 || D == 256, RA_ERR_UNSUPPORTED,
              "%s: unsupported head_dim=%d (supported: 32, 64, 128, 256)", what, D);
  RAB_REQUIRE(shape->batch >= 0 && shape->seq_q >= 0 && shape->seq_k >= 0, RA_ERR_INVALID, "%s: bad shape", what);
  RAB_REQUIRE(H > 0 && kvH > 0 && H % kvH == 0 && H <= 1 << 16, RA_ERR_INVALID, "%s: heads are a multiple of kv_heads", what);
  RAB_REQUIRE(shape->seq_q <= (1 << 30) && shape->seq_k <= (1 << 30), RA_ERR_INVALID, "%s: too many rows", what);
  // Blocks take the numbers of places without rows over one after the other, some 2.3 us each (32768 places with one sequence of 300 rows among them,
  // 8 KV heads: 2.0 ms), while their other warps wait: so many that this takes half a second of the 2 s that a wait may.
  RAB_REQUIRE(shape->batch <= (1 << 22) && static_cast<long long>(shape->batch) * H <= (1 << 25), RA_ERR_INVALID, "%s: too many sequences",
              what);
  if (shape->batch == 0 || shape->seq_q == 0) return RA_OK;
  RAB_REQUIRE(ends && q->data && out->data && (shape->seq_k == 0 || (k->data && v->data)), RA_ERR_INVALID, "%s: null argument", what);
  RAB_REQUIRE(((reinterpret_cast<uintptr_t>(ends) | reinterpret_cast<uintptr_t>(k_ends) | reinterpret_cast<uintptr_t>(lse)) & 3u) == 0,
              RA_ERR_INVALID, "%s: ends, k_ends or lse are not aligned to their elements", what);
  RAB_REQUIRE(rows_for_tma(*q, D, H, shape->seq_q) && rows_for_tma(*out, D, H, shape->seq_q), RA_ERR_INVALID,
              "%s: rows and heads must begin at multiples of 16 bytes and not overlap", what);
  RAB_REQUIRE(rows_apart(*out, D, H, shape->seq_q), RA_ERR_INVALID, "%s: rows of the result overlap", what);
  // without keys nothing is copied, but the maps want an address: the queries'
  const ra_rows none = {q->data, 0, D, static_cast<long long>(kvH) * D};
  const ra_rows& kr = shape->seq_k > 0 ? *k : none;
  const ra_rows& vr = shape->seq_k > 0 ? *v : none;
  RAB_REQUIRE(rows_for_tma(kr, D, kvH, shape->seq_k) && rows_for_tma(vr, D, kvH, shape->seq_k), RA_ERR_INVALID,
              "%s: rows and heads must begin at multiples of 16 bytes and not overlap", what);
  PackedArgs a;
  std::memset(&a, 0, sizeof(a));
  a.out = static_cast<char*>(out->data);
  a.out_row = out->row_stride;
  a.out_head = out->head_stride;
  a.lse = lse;
  a.ends = ends;
  a.k_ends = k_ends ? k_ends : ends;
  a.rows = shape->seq_q;
  a.k_rows = shape->seq_k;
  a.B = shape->batch;
  a.H = H;
  a.kvH = kvH;
  a.G = H / kvH;
  a.causal = causal != 0;
  a.status = device_status_ptr();
  RAB_REQUIRE(a.status != nullptr, RA_ERR_CUDA, "%s: no device status word", what);
  a.wait_ns = tc_wait_limit_ns();
  a.stall_after = tc_stall_after();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  auto go = [&](auto t) -> int {
    using T = decltype(t);
    if (D == 32) return launch_packed<64, 32, T>(*q, kr, vr, a, stream);
    if (D == 64) return launch_packed<64, 64, T>(*q, kr, vr, a, stream);
    if (D == 128) return launch_packed<128, 128, T>(*q, kr, vr, a, stream);
    return launch_packed<256, 256, T>(*q, kr, vr, a, stream);
  };
  return dtype == RA_BF16 ? go(__nv_bfloat16()) : go(__half());
}
