// kvc_prefill_q8_split.h -- the rule for the work split of a prefill launch over
// sequences with 8-bit blocks (host code without HIP, so that a test can
// compile it alone).
#pragma once

#include <algorithm>

#include "kvc_internal.h"

namespace kvc {

// Whether a launch runs as the bf16 prefill's variant instead, whose workgroups
// take 32 query rows: prefill_q8_kernel pads to 64, and its runs begin and end
// more slowly (8 us a run, 15-20 us for the fold of the cut items).  us, that
// variant / prefill_q8_kernel, bf16 out: 1 sequence over 4001 keys, 64 rows 30 /
// 45, 128 rows 34 / 57, 200 rows 51 / 53, 512 rows 76 / 73; 4 over 1000-4000, 64
// rows 37 / 51, 128 rows 60 / 58, 400 rows 167 / 113; 16 over 256-6000, 32 rows
// 63 / 78, 64 rows 101 / 94, 128 rows 228 / 165; 64 over 100-3000, 32 rows 143 /
// 158; 8 over 8000-16000, 32 rows 98 / 127, 128 rows 354 / 232.
inline bool prefill_q8_few(const PrefillArgs& a) {
    constexpr int64_t kMost = 2000;  // blocks of 64 rows and 32 keys
    if (a.n_q <= 32) return true;
    int64_t blocks = 0;
    for (int32_t j = 0; j < a.n_seqs; j++)
        for (int64_t r = 0; r < a.n_q && blocks <= kMost; r += kP8Rows)
            blocks += (a.q_pos0[j] + std::min<int64_t>(r + kP8Rows, a.n_q) + kBlockTok - 1) / kBlockTok * kKvHeads;
    return blocks <= kMost;
}

// Whether the line of a launch's key blocks has 32-bit indices with room to
// spare (every item counted as its sequence's longest): checked for a call's
// launches before the first one is made.
inline bool prefill_q8_fits(const PrefillArgs& a) {
    const int64_t n_rb = ((int64_t)a.n_q + kP8Rows - 1) / kP8Rows;
    int64_t total = 0;
    for (int32_t j = 0; j < a.n_seqs; j++)
        total += kKvHeads * n_rb * (((int64_t)a.q_pos0[j] + a.n_q + kBlockTok - 1) / kBlockTok);
    return total <= INT32_MAX / 2;
}

// Fills begin, cut, seq_at, n_wgs and per_xcd from n_seqs, n_q and q_pos0, for
// launches that fit.  A workgroup pays kP8Item blocks' time for
// each item that it takes up (its query rows, first copies and result) and a
// block's for each block; a cut inside an item costs two partials and their
// fold.  So runs are filled in order up to a common bound, an item that fits
// is not cut, and one that does not is cut only into parts of a fifth of the
// bound and more; the bound is raised until the runs are few enough.
inline void prefill_q8_split(PrefillQ8Args& a) {
    constexpr int64_t kP8Item = 7, kP8MinPart = 4;
    const auto blocks = [&](int32_t j, int64_t rb) {
        return (a.q_pos0[j] + std::min<int64_t>((rb + 1) * kP8Rows, a.n_q) + kBlockTok - 1) / kBlockTok;
    };
    const int64_t n_rb = (a.n_q + kP8Rows - 1) / kP8Rows;
    int64_t total = 0, longest = 0;
    for (int32_t j = 0; j < a.n_seqs; j++) {
        a.begin[j] = (int32_t)total;
        for (int64_t rb = 0; rb < n_rb; rb++) total += kKvHeads * blocks(j, rb);
        longest = std::max(longest, blocks(j, n_rb - 1));
    }
    a.begin[a.n_seqs] = (int32_t)total;
    const int64_t items = a.n_seqs * n_rb * kKvHeads;
    const auto fill = [&](int64_t bound) -> bool {
        const int64_t part = std::max(kP8MinPart, bound / 5);
        int32_t w = 0;
        int64_t load = 0, at = 0;
        const auto next = [&](int32_t j) {
            load = 0;
            if (++w >= kP8MaxWgs) return false;
            a.cut[w] = (int32_t)at;
            a.seq_at[w] = (uint8_t)j;
            return true;
        };
        a.cut[0] = 0;
        a.seq_at[0] = 0;
        for (int32_t j = 0; j < a.n_seqs; j++)
            for (int32_t h = 0; h < kKvHeads; h++)
                for (int64_t rb = 0; rb < n_rb; rb++) {
                    int64_t left = blocks(j, rb);
                    if (load && load + kP8Item + std::min(left, part) > bound && !next(j)) return false;
                    while (left > 0) {
                        const int64_t room = bound - load - kP8Item;
                        int64_t take = left;
                        if (left > room) {
                            take = std::max(room, part);
                            if (left - take < part) take = left >= 2 * part ? left - part : left;
                            if (load && take >= left) {  // too short to be cut here
                                if (!next(j)) return false;
                                continue;
                            }
                        }
                        load += kP8Item + take;
                        at += take;
                        left -= take;
                        if (left > 0 && !next(j)) return false;
                    }
                }
        a.n_wgs = w + 1;
        a.cut[w + 1] = (int32_t)at;
        return true;
    };
    int64_t bound = std::max<int64_t>(kP8Item + kP8MinPart, (total + kP8Item * items + kP8MaxWgs - 1) / kP8MaxWgs);
    while (!fill(bound)) bound += std::max<int64_t>(1, bound / 24);
    a.per_xcd = (a.n_wgs + 7) / 8;
    a.fold = 16;
}

}  // namespace kvc
