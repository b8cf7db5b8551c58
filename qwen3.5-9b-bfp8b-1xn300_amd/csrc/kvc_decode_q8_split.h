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
inline void decode_q8_split(const int32_t* nb, int32_t n, int32_t chunk_blocks, DecodeQ8Args& a) {
    int64_t total = 0;  // in 8-bit blocks; a bf16 block has the bytes of two
    for (int32_t j = 0; j < n; j++) total += a.n8[j] + 2 * (nb[j] - a.n8[j]);
    int32_t cb8 = chunk_blocks > 0 ? chunk_blocks : std::max(4, (int32_t)std::lround(0.25 * std::sqrt((double)total)));
    for (;; cb8 *= 2) {
        const int32_t cbf = chunk_blocks > 0 ? cb8 : std::max(2, cb8 / 2);
        int64_t chunks = 0;
        for (int32_t j = 0; j < n; j++) {
            a.chunk_begin[j] = (int32_t)chunks;
            chunks += (a.n8[j] + cb8 - 1) / cb8 + (nb[j] - a.n8[j] + cbf - 1) / cbf;
        }
        a.chunk_begin[n] = a.total_chunks = (int32_t)chunks;
        a.cb8 = cb8;
        a.cbf = cbf;
        if (chunks <= kMaxChunks) break;
    }
    a.n_items = a.total_chunks * kKvHeads;
    a.per_xcd = (a.n_items + 7) / 8;
}

}  // namespace kvc
