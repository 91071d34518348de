// Row blocks of a batch of sequences of different lengths: which sequence a
// workgroup's block belongs to, from `starts` alone.
#pragma once
#include "mix_types.h"

namespace rl {

// Sequence s has rows starts[s] .. starts[s + 1] (or row s, without starts) in blocks of `size`, its first block at number
// starts[s] / size + s: no two sequences begin at the same, each has at least one, and there are at most rows / size + seqs
// of them.
struct RowBlock {
    uint32_t seq, block; // the block's number in its sequence
    uint32_t begin, rows; // of the whole sequence, within the call's rows whatever `starts` holds
    bool used;
};

struct RowBlocks {
    uint32_t size, inv, next_inv; // inverse_of size, and of size + 1
};
inline RowBlocks row_blocks(uint32_t size) { return {size, inverse_of(size), inverse_of(size + 1)}; }
inline uint32_t row_block_count(uint32_t rows, uint32_t seqs, uint32_t size) { return rows / size + seqs; }

// Block b, found by the whole wave: 64 sequences a step, so one load's latency up to 64 sequences and two up to 4096.
__device__ inline RowBlock find_block(const int32_t *starts, uint32_t rows, uint32_t seqs, RowBlocks blocks, uint32_t b) {
    const auto start = [&](uint32_t i) { return (uint32_t)min(max(starts[i], 0), (int32_t)rows); };
    const auto number = [&](uint32_t row) { return split_by(row, blocks.size, blocks.inv).x; };
    const uint32_t lane = threadIdx.x % 64;
    RowBlock r{0, 0, 0, 0, false};
    if (!starts) { // one row a sequence, its block at i / size + i: every size-th number is none's
        r.seq = b - split_by(b, blocks.size + 1, blocks.next_inv).x;
        if (number(r.seq) + r.seq != b || r.seq >= seqs) return r;
        r.begin = r.seq, r.rows = 1, r.used = true;
        return r;
    }
    uint32_t lo = 0;
    for (uint32_t n = seqs; n > 1;) {
        const uint32_t step = (n + 63) / 64, at = lane * step;
        const bool before = at < n && number(start(lo + (at < n ? at : 0))) + lo + at <= b;
        const uint32_t count = (uint32_t)__popcll(__ballot(before));
        if (count == 0) return r;
        lo += (count - 1) * step;
        n = min(step, n - (count - 1) * step);
    }
    r.seq = __builtin_amdgcn_readfirstlane(lo);
    r.begin = start(r.seq);
    r.rows = max((int32_t)start(r.seq + 1) - (int32_t)r.begin, 0);
    const uint32_t first = number(r.begin) + r.seq;
    r.block = b - first;
    r.used = first <= b && (r.block == 0 || (uint64_t)r.block * blocks.size < r.rows);
    return r;
}

}  // namespace rl
