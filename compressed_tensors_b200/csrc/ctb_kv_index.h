// Index arithmetic of the paged cache, for the kernels and for a host test: every value that comes from device memory
// (row offsets, lengths, block numbers) is brought into the range that the buffers have before it is used as an index.
#pragma once

#include <stdint.h>

#include "../../include/ctb200.h"

#ifdef __CUDACC__
#define CTB_HD __host__ __device__ __forceinline__
#else
#define CTB_HD inline
#endif

namespace ctb {

struct KvSeq {
    int first_row, rows;  // rows of the token-major inputs that belong to the request
    int len;              // cached tokens, those rows included, no more than the block table can hold
    int start;            // position of the first row; below zero where there are more rows than tokens
};

CTB_HD KvSeq kv_seq(int64_t lo, int64_t hi, int64_t len, int64_t tokens, int64_t capacity) {
    KvSeq s;
    const int64_t a = lo < 0 ? 0 : (lo > tokens ? tokens : lo), z = hi > tokens ? tokens : hi;
    if (len < 0) len = 0;
    s.first_row = (int)a;
    s.rows = (int)(z > a ? z - a : 0);
    s.start = (int)(len - s.rows);
    s.len = (int)(len > capacity ? capacity : len);
    return s;
}

// Blocks of a request that its rows are written to: the first one, and how many.
CTB_HD int kv_written_blocks(const KvSeq &s, int block_size, int &first_block) {
    const int lo = s.start < 0 ? 0 : s.start;
    first_block = lo / block_size;
    return s.rows > 0 && s.len > lo ? (s.len - 1) / block_size - first_block + 1 : 0;
}

// An upper bound of the blocks that a call writes, known without the lengths: each holds at least one of the rows, and
// a request fills all but two of those that it writes.
CTB_HD int64_t kv_most_written(int64_t tokens, int64_t batch, int64_t block_size) {
    const int64_t fill = tokens / block_size + 2 * batch;
    return tokens < fill ? tokens : fill;
}

// The positions that row i of a request sees: [0, kv_end).
CTB_HD int kv_end(const KvSeq &s, int64_t i, bool causal) {
    if (!causal) return s.len;
    const int64_t e = (int64_t)s.start + i + 1;
    return (int)(e < 0 ? 0 : (e < s.len ? e : s.len));
}

}  // namespace ctb
