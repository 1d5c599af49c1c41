// Rows of K and V to a paged cache in 4 bits, with their norm and rotation and the queries of the same tokens, as paged_append has them
// for a cache in 16 and 32 bits: the same kernel (norm_rope.cuh) with another way out. It is bound by the rows that come in, at two
// bytes an element, and 9 / 16 of one go out.
#include "norm_rope.cuh"

using namespace rab;

extern "C" {

int ra_paged_append_4bit(const ra_paged_kv* cache, float k_scale, float v_scale, const ra_rows* k, const ra_rows* v, int rows,
                         const int* counts, const ra_rows* q, const ra_rows* q_out, int heads, const ra_norm_rope* how,
                         ra_stream stream) {
  return append_rows<true>("paged_append_4bit", cache, k, v, rows, counts, q, q_out, heads, how, k_scale, v_scale, stream);
}

}  // extern "C"
