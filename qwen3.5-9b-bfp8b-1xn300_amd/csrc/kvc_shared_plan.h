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
    int32_t listed = 0;                // of them in nodes of several, each filled up to a multiple of 8
    int32_t n_items = 0;               // workgroups
    int32_t parts = 0;                 // partials per q head, of all sequences
    int32_t path = 0;                  // most of them of one sequence
    int32_t group = kSharedSeqs;       // members of a workgroup: 4 (a tile) or 8
    int64_t blocks = 0, blocks_apart = 0;  // read by the plan, and sequence by sequence
    int64_t tile_work = 0;             // blocks of a kv head for up to kSharedSeqs members
    int32_t first[kSharedNodes];       // of the node's blocks, in its members' tables
    int32_t len[kSharedNodes];         // blocks
    int32_t item_begin[kSharedNodes + 1];
    uint16_t chunk[kSharedNodes];      // blocks per workgroup
    uint16_t member_begin[kSharedNodes];
    uint8_t members[kSharedNodes];
    uint8_t kind[kSharedNodes];
    uint8_t member[kSharedMembers + kMaxBatch];  // index of the sequence in the launch
    uint16_t part[kSharedMembers + kMaxBatch];   // its first partial of this node
    int32_t seq_row[kMaxBatch];        // its first partial in the workspace
    int32_t seq_parts[kMaxBatch];
};

// A node is worth its own partials from this many saved block reads on.
constexpr int32_t kSharedMinSaved = 4;

class SharedPlanner {
  public:
    // tab[i]: block ids of sequence i; keys[i]: keys attended (0 allowed)
    SharedPlanner(const int32_t* const* tab, const int32_t* keys, int32_t n, SharedPlan& p) : tab_(tab), keys_(keys), p_(p) {
        p_.n_nodes = p_.n_members = p_.listed = 0;
        p_.blocks = p_.blocks_apart = 0;
        for (int32_t i = 0; i < n; i++) {
            order_[i] = (uint8_t)i;
            p_.blocks_apart += total(i);
        }
        walk(0, n, 0, 0);
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
        p_.members[k] = (uint8_t)(hi - lo);
        for (int32_t i = lo; i < hi; i++) p_.member[p_.n_members++] = order_[i];
        p_.blocks += to - from;
        if (hi - lo > 1) p_.listed += (hi - lo + kSharedSeqs - 1) / kSharedSeqs * kSharedSeqs;
    }

    // order_[lo, hi) run together up to block `at`; their blocks from `from` on
    // (<= at) have no node yet.
    void walk(int32_t lo, int32_t hi, int32_t from, int32_t at) {
        if (hi - lo == 1) {
            if (total(order_[lo]) > from) emit(lo, hi, from, total(order_[lo]));
            return;
        }
        int32_t end = full(order_[lo]);
        for (int32_t i = lo + 1; i < hi; i++)
            end = common(order_[lo], order_[i], at, std::min(end, full(order_[i])));
        if ((int64_t)(end - from) * (hi - lo - 1) >= kSharedMinSaved && p_.listed + (hi - lo + kSharedSeqs - 1) / kSharedSeqs * kSharedSeqs <= kSharedMembers) {
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
};

inline int32_t shared_groups(const SharedPlan& p, int32_t members) { return (members + p.group - 1) / p.group; }

// Nodes of several members first, then the long ones: what runs last is short.
inline void shared_sort(SharedPlan& p) {
    uint8_t order[kSharedNodes];
    for (int32_t k = 0; k < p.n_nodes; k++) order[k] = (uint8_t)k;
    const SharedPlan was = p;
    std::sort(order, order + p.n_nodes, [&](uint8_t a, uint8_t b) {
        const bool x = was.members[a] > 1, y = was.members[b] > 1;
        return x != y ? x : was.len[a] != was.len[b] ? was.len[a] > was.len[b] : a < b;
    });
    for (int32_t k = 0; k < p.n_nodes; k++) {
        p.first[k] = was.first[order[k]];
        p.len[k] = was.len[order[k]];
        p.member_begin[k] = was.member_begin[order[k]];
        p.members[k] = was.members[order[k]];
    }
}

// Cuts the nodes into workgroups: of several members, up to `halves` half blocks a
// wave (a node that has no more goes to workgroups that take all kv heads), of one
// member `one` blocks each.
inline void shared_items(SharedPlan& p, int32_t halves, int32_t one, int32_t n) {
    for (int32_t i = 0; i < n; i++) p.seq_parts[i] = 0;
    int64_t items = 0;
    for (int32_t k = 0; k < p.n_nodes; k++) {
        const int32_t members = p.members[k], groups = shared_groups(p, members);
        p.kind[k] = members == 1 ? kSharedOne : 2 * p.len[k] <= halves ? kSharedHeads : kSharedKeys;
        int32_t chunk = members == 1 ? one : p.kind[k] == kSharedHeads ? p.len[k] : 2 * halves;
        int32_t n_chunks = (p.len[k] + chunk - 1) / chunk;
        // equal ones, of whole rounds of the 4 waves
        chunk = (p.len[k] + n_chunks - 1) / n_chunks;
        if (p.kind[k] == kSharedKeys) chunk = (chunk + 1) / 2 * 2;
        n_chunks = (p.len[k] + chunk - 1) / chunk;
        const int32_t units = n_chunks * (p.kind[k] == kSharedHeads ? 1 : kKvHeads);
        p.chunk[k] = (uint16_t)chunk;
        // (the groups of a unit run on one XCD: such nodes start on a multiple of 8)
        if (groups > 1) items = (items + 7) / 8 * 8;
        p.item_begin[k] = (int32_t)items;
        items += groups > 1 ? (int64_t)(units + 7) / 8 * 8 * groups : units;
        for (int32_t i = p.member_begin[k]; i < p.member_begin[k] + members; i++) {
            p.part[i] = (uint16_t)std::min(p.seq_parts[p.member[i]], kSharedPath);
            p.seq_parts[p.member[i]] += n_chunks;
        }
    }
    p.item_begin[p.n_nodes] = (int32_t)items;
    p.n_items = (int32_t)items;
    p.path = 0;
    int64_t parts = 0;
    for (int32_t i = 0; i < n; i++) {
        p.seq_row[i] = (int32_t)parts;
        parts = std::min<int64_t>(parts + p.seq_parts[i], INT32_MAX);
        p.path = std::max(p.path, p.seq_parts[i]);
    }
    p.parts = (int32_t)parts;
}

// Whether the partials fit.
inline bool shared_fits(const SharedPlan& p) { return p.path <= kSharedPath && p.parts <= kSharedMaxParts; }

// Whether the plan beats kvc_decode_attn's launch, by the us that either takes: a
// fixed part (here two launches, the first longer for more members), blocks from
// memory, blocks that sequence by sequence come from the caches, and the tiles' LDS.
// us per layer, kvc_decode_attn / shared (profiles/shared_decode_rule.txt): 4 sequences on
// 300 tokens 8.9 / 12.2, 2 on 4096 11.6 / 12.8, 4 on 4096 13.4 / 13.5, 8 on 1000 9.1 / 12.3,
// 8 on 2000 11.3 / 12.3, 8 on 4096 17.9 / 13.7, 16 on 1000 11.5 / 12.5, 16 on 2000 16.5 /
// 12.4, 64 on 2000 46.5 / 17.9, 64 with 96 tokens in common of 1031 45.5 / 47.2, 64 on
// 65536 1229 / 139.
// `always`: wherever blocks are shared.
inline bool shared_pays(const SharedPlan& p, int32_t n, bool always) {
    if (!shared_fits(p) || p.blocks == p.blocks_apart) return false;
    if (always) return true;
    constexpr double kBlockUs = 2.0 * kBlockBytes * 1e-6;  // of a block, K and V, at 1 TB/s
    const double shared = 6.8 + std::min(0.6 * n, 5.7) + std::max(p.blocks * kBlockUs / 5.5, 0.002 * p.tile_work);
    const double apart = 7 + std::max(p.blocks * kBlockUs / 6.5, p.blocks_apart * kBlockUs / 12);
    return shared < apart;
}

// Blocks of all kv heads that workgroups read in nodes of one member [0] and of
// several [1].
inline void shared_work(const SharedPlan& p, int64_t* work) {
    work[0] = work[1] = 0;
    for (int32_t k = 0; k < p.n_nodes; k++)
        work[p.members[k] > 1] += (int64_t)p.len[k] * kKvHeads * shared_groups(p, p.members[k]);
}

// The work of a launch of n sequences (n <= kMaxBatch): caller_chunk > 0 is a
// chunk length that the caller set.  Otherwise nodes of several members and of one
// are each cut into about a workgroup per CU.  (Two fit, but those on tiles then
// share its LDS and take twice the time, and shorter chunks leave more partials to
// fold.)
//
// Groups of 4 members are one tile: half of the registers, of the fold of the waves
// and of the work of a chunk, and the blocks are read from L2 twice as often.  That
// pays for nodes of up to 8 and in small launches; us per layer in groups of 4 / 8: 8
// sequences on 4096 tokens 14.9 / 16.0, 16 on 2000 13.5 / 14.9, 32 on 4096 18.7 / 21.3,
// 8 on 32768 34.4 / 36.9; 64 on 4096 23.8 / 22.4, 64 on 8192 62 / 58, 16 on 65536 83 /
// 63.  Chunks of 8 blocks at least (4, 8 and 12 blocks: 16 on 2000 15.6, 13.5, 14.0), or
// of 12 where those of three and more groups nearly fill the GPU (8 and 12: 16 on 4096
// 16.0, 14.4; 12 on 3000 13.7, 13.7; but 8 on 8192, in two groups, 16.7, 18.1).
inline void shared_plan(const int32_t* const* tab, const int32_t* keys, int32_t n, int32_t caller_chunk, SharedPlan& p) {
    SharedPlanner(tab, keys, n, p);
    shared_sort(p);
    int64_t work[2];
    p.group = kSharedSeqs;
    shared_work(p, work);
    p.tile_work = work[1];
    int32_t most = 0;
    for (int32_t k = 0; k < p.n_nodes; k++) most = std::max<int32_t>(most, p.members[k]);
    p.group = kSharedTile;
    shared_work(p, work);
    if (most > kSharedSeqs && work[1] > 16 * kSharedCus) {
        p.group = kSharedSeqs;
        shared_work(p, work);
    }
    const auto per_cu = [](int64_t w, int64_t least) { return std::max(least, (w + kSharedCus - 1) / kSharedCus); };
    const int64_t tiles = caller_chunk > 0 ? caller_chunk : per_cu(work[1], most > kSharedSeqs && work[1] > 6 * kSharedCus ? 12 : 8);
    int32_t halves = (int32_t)std::min<int64_t>(kSharedHalves, (tiles + 1) / 2);
    int32_t one = (int32_t)std::min<int64_t>(kSharedOneMax, caller_chunk > 0 ? caller_chunk : per_cu(work[0], 3));
    shared_items(p, halves, one, n);
    while (!shared_fits(p) && (halves < kSharedHalves || one < kSharedOneMax)) {
        halves = std::min(2 * halves, kSharedHalves);
        one = std::min(2 * one, kSharedOneMax);
        shared_items(p, halves, one, n);
    }
}

}  // namespace kvc
