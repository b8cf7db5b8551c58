// kvc_decode_q8_split.h -- the rule for the work split of a decode launch over
// sequences with 8-bit blocks (host code without HIP, so that a test can
// compile it alone).
#pragma once

#include <algorithm>
#include <cmath>

#include "kvc_internal.h"

namespace kvc {

// Chunk lengths (a.cb8 8-bit blocks, a.cbf bf16 blocks), the sequences' first
// chunks and the launch's items, from the block counts nb[n] and a.n8.
// chunk_blocks: the caller's choice for both (kvc_config), 0 = automatic.
//
// A chunk is 4 workgroups (one per kv head) of 4 waves, so 96 chunks are 1.5
// workgroups per CU: below that more chunks win, and the loop takes the
// shortest multiple of 4 blocks that stays within it, up to 20 or to one chunk
// per sequence.  Above it a chunk's start, exchange and combine weigh more
// than the tail of the last workgroups; both shrink the total relatively with
// the square root of the launch.  us per layer of calls back to
// back, this rule / chunks of:
//   1 x 4096 tokens        9.0 / 8: 10.7
//   1 x 16000             14.3 / 8: 14.5
//   2 x 6000              12.7 / 8: 12.2, 12: 13.3
//   4 x 3000..9000        18.6 / 8: 17.4, 16: 17.5
//   8 x 777..6001         20.5 / 8: 22.4, 16: 22.0
//   64 x 300              18.6 / 4: 22.7
//   24 x 100..4000        29.5 / 8: 28.3, 16: 26.4
//   64 x 500..3000        58.7 / 8: 58.8, 12: 57.0, 24: 57.8
//   64 x 512..16384      178.0 / 16: 188.5, 24: 183.3, 32: 180.1, 48: 186.6
// (behind the best fixed length by up to 11 % between those ends)
inline void decode_q8_split(const int32_t* nb, int32_t n, int32_t chunk_blocks, DecodeQ8Args& a) {
    int64_t total = 0;  // in 8-bit blocks; a bf16 block has the bytes of two
    int32_t longest = 1;
    for (int32_t j = 0; j < n; j++) {
        total += a.n8[j] + 2 * (nb[j] - a.n8[j]);
        longest = std::max(longest, a.n8[j]);
    }
    int32_t cb8 = 0, cbf = 0;
    const auto cut = [&](int32_t cb) {
        cb8 = cb;
        // a bf16 block has twice the bytes, an 8-bit one more instructions per byte
        cbf = chunk_blocks > 0 ? cb : std::max(4, cb * 2 / 3);
        int64_t chunks = 0;  // 64 bits: a caller's chunk of 1 block
        for (int32_t j = 0; j < n; j++) {
            a.chunk_begin[j] = (int32_t)chunks;
            chunks += (a.n8[j] + cb8 - 1) / cb8 + (nb[j] - a.n8[j] + cbf - 1) / cbf;
        }
        a.chunk_begin[n] = (int32_t)chunks;
        return chunks;
    };
    int64_t chunks;
    if (chunk_blocks > 0) {
        chunks = cut(caller_chunk_blocks(chunk_blocks));
    } else {
        for (cb8 = 4; (chunks = cut(cb8)) > 96 && cb8 < std::min(longest, 20); cb8 += 4) {}
        if (chunks > 96) chunks = cut(std::max(12, (int32_t)std::lround(0.25 * std::sqrt((double)total))));
    }
    while (chunks > kMaxChunks) chunks = cut(2 * cb8);
    a.cb8 = cb8;
    a.cbf = cbf;
    a.total_chunks = (int32_t)chunks;
    a.n_items = a.total_chunks * kKvHeads;
    a.per_xcd = (a.n_items + 7) / 8;
}

}  // namespace kvc
