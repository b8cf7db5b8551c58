// kvc_shared_plan.h -- how a decode launch over sequences that share blocks is
// cut into work (host code without HIP, so that a test can compile it alone).
//
// The sequences' block tables form a trie: two sequences run together as long
// as their tables name the same blocks.  A node is a run of blocks and the
// sequences (members) that all attend it; the nodes on a sequence's path cover
// its blocks once, in order.  Shared nodes hold only blocks that are full for
// every member, so that no key of one is hidden from one member and seen by
// another; what is left of a sequence is a node of its own.
#pragma once

#include <algorithm>
#include <cstring>

#include "kvc_internal.h"

namespace kvc {

struct SharedPlan {
    int32_t n_nodes = 0, n_members = 0;
    int32_t n_items = 0;               // workgroups
    int32_t rows = 0;                  // partial rows
    int32_t path = 0;                  // most partials of one (sequence, q head)
    int64_t blocks = 0, blocks_apart = 0;  // read by the plan, and sequence by sequence
    int32_t first[kSharedNodes];       // of the node's blocks, in its members' tables
    int32_t len[kSharedNodes];         // blocks
    int32_t item_begin[kSharedNodes + 1];
    int32_t row_begin[kSharedNodes];
    uint16_t chunk[kSharedNodes];      // blocks per workgroup
    uint16_t member_begin[kSharedNodes + 1];
    uint8_t kind[kSharedNodes];
    uint8_t member[kSharedMembers];    // index of the sequence in the launch
};

// A node is worth its own partials from this many saved block reads on.
constexpr int32_t kSharedMinSaved = 4;

class SharedPlanner {
  public:
    // tab[i]: block ids of sequence i; keys[i]: keys attended (0 allowed)
    SharedPlanner(const int32_t* const* tab, const int32_t* keys, int32_t n, SharedPlan& p) : tab_(tab), keys_(keys), p_(p) {
        p_.n_nodes = p_.n_members = 0;
        p_.blocks = p_.blocks_apart = 0;
        for (int32_t i = 0; i < n; i++) {
            order_[i] = (uint8_t)i;
            p_.blocks_apart += total(i);
        }
        left_ = n;
        walk(0, n, 0, 0);
        p_.member_begin[p_.n_nodes] = (uint16_t)p_.n_members;
    }

  private:
    int32_t total(int32_t s) const { return (keys_[s] + kBlockTok - 1) / kBlockTok; }
    int32_t full(int32_t s) const { return keys_[s] / kBlockTok; }

    // First index in [at, end) where the tables differ, or end.
    int32_t common(int32_t a, int32_t b, int32_t at, int32_t end) const {
        const int32_t *x = tab_[a], *y = tab_[b];
        while (at + 16 <= end && memcmp(x + at, y + at, 64) == 0) at += 16;
        while (at < end && x[at] == y[at]) at++;
        return at;
    }

    void emit(int32_t lo, int32_t hi, int32_t from, int32_t to) {
        const int32_t k = p_.n_nodes++;
        p_.first[k] = from;
        p_.len[k] = to - from;
        p_.member_begin[k] = (uint16_t)p_.n_members;
        for (int32_t i = lo; i < hi; i++) p_.member[p_.n_members++] = order_[i];
        p_.blocks += to - from;
    }

    // order_[lo, hi) run together up to block `at`; their blocks from `from` on
    // (<= at) have no node yet.
    void walk(int32_t lo, int32_t hi, int32_t from, int32_t at) {
        if (hi - lo == 1) {
            left_--;
            if (total(order_[lo]) > from) emit(lo, hi, from, total(order_[lo]));
            return;
        }
        int32_t end = full(order_[lo]);
        for (int32_t i = lo + 1; i < hi; i++)
            end = common(order_[lo], order_[i], at, std::min(end, full(order_[i])));
        // (a leaf for each sequence that has none yet still has to fit)
        if ((int64_t)(end - from) * (hi - lo - 1) >= kSharedMinSaved && p_.n_members + (hi - lo) + left_ <= kSharedMembers) {
            emit(lo, hi, from, end);
            from = end;
        }
        // groups that go on with the same full block; the others go on alone
        for (int32_t i = lo; i < hi;) {
            const int32_t s = order_[i];
            int32_t j = i + 1;
            if (full(s) > end)
                for (int32_t k = j; k < hi; k++)
                    if (full(order_[k]) > end && tab_[order_[k]][end] == tab_[s][end]) {
                        std::rotate(order_ + j, order_ + k, order_ + k + 1);
                        j++;
                    }
            walk(i, j, from, end);
            i = j;
        }
    }

    const int32_t* const* tab_;
    const int32_t* keys_;
    SharedPlan& p_;
    uint8_t order_[kMaxBatch];
    int32_t left_ = 0;  // sequences without a leaf
};

inline int32_t shared_groups(int32_t members) { return (members + kSharedSeqs - 1) / kSharedSeqs; }

// Items of the nodes, for the chunk length c (blocks of a workgroup).
inline void shared_items(SharedPlan& p, int32_t c, int32_t n) {
    int32_t chunks_of[kMaxBatch] = {};
    int64_t items = 0, rows = 0;
    for (int32_t k = 0; k < p.n_nodes; k++) {
        const int32_t members = p.member_begin[k + 1] - p.member_begin[k], groups = shared_groups(members);
        int32_t chunk;
        if (members > 4) {
            p.kind[k] = kSharedRows;
            chunk = std::min(c, kSharedMaxChunk);
        } else if (p.len[k] <= kSharedShort) {
            p.kind[k] = kSharedHeads;
            chunk = p.len[k];
        } else {
            p.kind[k] = kSharedKeys;
            chunk = std::min((c + 3) / 4 * 4, 4 * kSharedMaxChunk);
        }
        const int32_t n_chunks = (p.len[k] + chunk - 1) / chunk;
        p.chunk[k] = (uint16_t)chunk;
        p.item_begin[k] = (int32_t)items;
        p.row_begin[k] = (int32_t)rows;
        if (groups > 1)
            items += (int64_t)(n_chunks * kKvHeads + 7) / 8 * 8 * groups;
        else
            items += p.kind[k] == kSharedHeads ? n_chunks : n_chunks * kKvHeads;
        // (nodes of one group start anywhere, those of several on a multiple of 8)
        if (k + 1 < p.n_nodes && p.member_begin[k + 2] - p.member_begin[k + 1] > kSharedSeqs) items = (items + 7) / 8 * 8;
        rows += (int64_t)n_chunks * kQHeads * members;
        for (int32_t i = p.member_begin[k]; i < p.member_begin[k + 1]; i++) chunks_of[p.member[i]] += n_chunks;
    }
    p.item_begin[p.n_nodes] = (int32_t)items;
    p.n_items = (int32_t)items;
    p.rows = (int32_t)std::min<int64_t>(rows, INT32_MAX);
    p.path = 0;
    for (int32_t i = 0; i < n; i++) p.path = std::max(p.path, chunks_of[i]);
}

// Whether the plan beats reading sequence by sequence, and fits.
inline bool shared_pays(const SharedPlan& p) {
    return p.path <= kSharedPath && p.rows <= kSharedMaxRows && p.blocks_apart - p.blocks >= 16;
}

// The work of a launch of n sequences (n <= kMaxBatch): caller_chunk > 0 is a
// chunk length that the caller set.
inline void shared_plan(const int32_t* const* tab, const int32_t* keys, int32_t n, int32_t caller_chunk, SharedPlan& p) {
    SharedPlanner(tab, keys, n, p);
    int64_t work = 0;
    for (int32_t k = 0; k < p.n_nodes; k++)
        work += (int64_t)p.len[k] * shared_groups(p.member_begin[k + 1] - p.member_begin[k]) * kKvHeads;
    int32_t c = caller_chunk > 0 ? std::min(caller_chunk, 4 * kSharedMaxChunk) : (int32_t)std::max<int64_t>(2, (work + 255) / 256);
    for (;;) {
        shared_items(p, c, n);
        if ((p.path <= kSharedPath && p.rows <= kSharedMaxRows) || c >= 4 * kSharedMaxChunk) break;
        c *= 2;
    }
}

}  // namespace kvc
