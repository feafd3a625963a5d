// Host build of the paged cache's index arithmetic (ctb_kv_index.h), called by test_serving_host.py.
#include "../compressed_tensors_b200/csrc/ctb_kv_index.h"

extern "C" {
void seq(int64_t lo, int64_t hi, int64_t len, int64_t tokens, int64_t capacity, int32_t *out) {
    const ctb::KvSeq s = ctb::kv_seq(lo, hi, len, tokens, capacity);
    out[0] = s.first_row, out[1] = s.rows, out[2] = s.len, out[3] = s.start;
}
int written(int64_t lo, int64_t hi, int64_t len, int64_t tokens, int64_t capacity, int block_size, int *first) {
    return ctb::kv_written_blocks(ctb::kv_seq(lo, hi, len, tokens, capacity), block_size, *first);
}
int64_t most_written(int64_t tokens, int64_t batch, int64_t block_size) { return ctb::kv_most_written(tokens, batch, block_size); }
int seen(int64_t lo, int64_t hi, int64_t len, int64_t tokens, int64_t capacity, int64_t i, int causal) {
    return ctb::kv_end(ctb::kv_seq(lo, hi, len, tokens, capacity), i, causal != 0);
}
}
