// Row blocks of a batch of sequences of different lengths: which sequence a
// workgroup's block belongs to, from `starts` alone.
#pragma once
#include "mix_types.h"

namespace rl {

// Sequence s has rows starts[s] .. starts[s + 1] (or row s, without starts) in blocks of 2^shift, its first block at
// number (starts[s] >> shift) + s: no two sequences begin at the same, each has at least one, and there are at most
// (rows >> shift) + seqs of them.
struct RowBlock {
    uint32_t seq, block; // the block's number in its sequence
    uint32_t begin, rows; // of the whole sequence, within the call's rows whatever `starts` holds
    bool used;
};

inline uint32_t row_blocks(uint32_t rows, uint32_t seqs, uint32_t shift) { return (rows >> shift) + seqs; }

// Block b, found by the whole wave: 64 sequences a step, so one load's latency up to 64 sequences and two up to 4096.
__device__ inline RowBlock find_block(const int32_t *starts, uint32_t rows, uint32_t seqs, uint32_t shift, uint32_t b) {
    const auto start = [&](uint32_t i) { return (uint32_t)min(max(starts[i], 0), (int32_t)rows); };
    const uint32_t lane = threadIdx.x % 64;
    RowBlock r{0, 0, 0, 0, false};
    if (!starts) { // one row a sequence
        const uint32_t whole = (1u << shift) - 1; // blocks (i >> shift) + i: every 2^shift-th number is none's
        r.seq = b - b / (whole + 2);
        if ((r.seq >> shift) + r.seq != b || r.seq >= seqs) return r;
        r.begin = r.seq, r.rows = 1, r.used = true;
        return r;
    }
    uint32_t lo = 0;
    for (uint32_t n = seqs; n > 1;) {
        const uint32_t step = (n + 63) / 64, at = lane * step;
        const bool before = at < n && (start(lo + (at < n ? at : 0)) >> shift) + lo + at <= b;
        const uint32_t count = (uint32_t)__popcll(__ballot(before));
        if (count == 0) return r;
        lo += (count - 1) * step;
        n = min(step, n - (count - 1) * step);
    }
    r.seq = __builtin_amdgcn_readfirstlane(lo);
    r.begin = start(r.seq);
    r.rows = max((int32_t)start(r.seq + 1) - (int32_t)r.begin, 0);
    const uint32_t first = (r.begin >> shift) + r.seq;
    r.block = b - first;
    r.used = first <= b && (r.block == 0 || (uint64_t)r.block << shift < r.rows);
    return r;
}

}  // namespace rl
