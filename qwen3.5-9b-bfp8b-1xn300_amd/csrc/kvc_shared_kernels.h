// kvc_shared_kernels.h -- decode attention for sequences that share blocks, each
// shared block read once (included by kvc_kernels.hip).
//
// For every trie node (kvc_shared_plan.h) of several members and kv head, the
// members' query rows (4 q heads each, 4 members to a tile of 16 rows) attend to the
// node's keys in one product per tile:
//   S^T[16 keys x 16 rows]  = K[keys x 256] . Q^T        (v_mfma_f32_16x16x32_bf16)
//   P^T = 2^(S^T - m), m the running maximum of the row
//   O^T[256 x 16 rows]     += V^T[256 x keys] . P^T      (v_mfma_f32_16x16x16_bf16)
// in the operand layouts of the prefill kernel: a lane stays on one row in both
// products, P^T leaves the accumulator in operand order, and V^T fragments come
// from LDS through the transposing read.  Every wave streams half blocks (16 keys)
// of its own through LDS units of its own, without barriers, for all tiles of its
// members, so a K or V fragment is read from LDS once for up to 32 rows, and two
// workgroups fit on a CU: while waves of one wait for a copy or fold, the other's
// run.  A second launch folds the partials (m, l, O) of a row: O = sum 2^(m_p - M)
// O_p, l likewise, and divides.  (A fold by the last workgroup to arrive, as
// kvc_decode_attn does it, would put all members of a group on one workgroup.)
//
// Measured, us per layer with bf16 output (kvc_decode_attn beside it): 8 sequences on
// 4096 common tokens 14.5 (17.6): this launch 10.2, one trip after the other to the
// arguments (0.8), the block ids and queries (1.1), the keys (3.9, at 5 TB/s: twice the
// half blocks in flight took 15.0) and the fold of the waves (1.5); the second launch
// 4.2.  64 on 8192, with tails of up to 1500 58 (194): this launch 54.6 for
// 240 MB from HBM, most of them the tails', the products 5 of it.  64 on 65536 139 (1229):
// bound by the blocks' eight trips from L2 to LDS.  30 in a tree of prompts, fp32 output
// 22.5 (36).
#pragma once

namespace kvc {

constexpr int kSharedTok = 16;  // keys of a unit: half a block
struct SharedSmem {
    // (K, V) units of each wave: rows of 512 B, 16-B chunks swizzled by the row (kswz, vswz)
    uint16_t unit[2 * kWaves][kSharedTok * kHeadDim];
    float2 ml[kWaves][16];
};
constexpr int kShAhead = 3;  // operand fragments read ahead of their MFMAs
constexpr uint32_t kUnitLds = kSharedTok * kHeadDim * 2;
typedef short bf16x4_t __attribute__((ext_vector_type(4)));  // (the 16x16x16 product's operand type)

template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

struct SharedOneSmem {
    DecodeSmem d;
    __align__(16) float p[kWaves][32];  // a block's weights of 8 tokens and 4 heads
};

// One workgroup's work: a chunk of a node for up to kSharedSeqs of its members.
struct SharedItem {
    int kind, h, ck, members;
    int keys;             // of the chunk
    const int32_t* trow;  // of its first block
    uint32_t who[4];      // the members' entries, two a word
};

// T: 16-row tiles; PARTS: bf16 parts of a weight (1 for bf16 output, 3 = 24 bits for fp32 output)
template <int T, int PARTS>
__device__ __forceinline__ void shared_item(const SharedArgs& a, const SharedItem& it, int seq_row, SharedSmem& sm) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q4 = lane >> 4, r16 = lane & 15;
    const int step = it.kind == kSharedKeys ? kWaves : 1, base = it.kind == kSharedKeys ? wave : 0;
    const int h = it.h;
    // block ids: lane i holds that of this wave's i-th half block
    const int n_half = it.keys / kSharedTok;  // (whole blocks)
    const int n_my = it.kind == kSharedKeys ? (n_half - wave + kWaves - 1) / kWaves : n_half;
    const int idv = lane < n_my ? it.trow[(base + lane * step) >> 1] : 0;

    // this lane's rows: member 4 t + r16 / 4, q head r16 % 4
    const int g = r16 & 3;
    const float c = fabsf(a.scale_log2);
    const uint32_t qflip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    const auto entry = [&](int t) { return (((r16 & 8) ? it.who[2 * t + 1] : it.who[2 * t]) >> ((r16 & 4) * 4)) & 0xFFFF; };
    bf16x8_t qb[T][8];
    {
        u32x4 x[T][8];
#pragma unroll
        for (int t = 0; t < T; t++) {
            const uint16_t* qr = a.q + ((size_t)(entry(t) & 63) * kQHeads + h * kGroup + g) * kHeadDim;
#pragma unroll
            for (int ks = 0; ks < 8; ks++) x[t][ks] = *reinterpret_cast<const u32x4*>(qr + 32 * ks + 8 * q4);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < T; t++)
#pragma unroll
            for (int ks = 0; ks < 8; ks++) {
#pragma unroll
                for (int i = 0; i < 4; i++) x[t][ks][i] ^= qflip;
                // waited for here, before the copies are issued: a later wait would
                // cover those too (8 sequences on 65536 tokens 58.9 us a layer, with
                // the wait behind the first copies 62.8)
                asm volatile("" : "+v"(x[t][ks]));
                qb[t][ks] = as_bf16x8(x[t][ks]);
            }
    }

    // copy p of a unit: rows 2p, 2p + 1; lane l fills position l % 32
    const uint32_t cbk = (((lane & 31) ^ (lane >> 5)) << 4) + (lane >> 5) * 512;
    const uint32_t cbv = (((lane & 31) ^ ((lane >> 5) << 1)) << 4) + (lane >> 5) * 512;
    auto issue = [&](const uint16_t* pool, uint32_t cb, int jsh, int i, uint32_t lds) {
        const int id = __builtin_amdgcn_readlane(idv, i);
        const int half = (base + i * step) & 1;
        const uint16_t* src = pool + (((size_t)id * kKvHeads + h) * kBlockTok + half * kSharedTok) * kHeadDim;
#pragma unroll
        for (int p = 0; p < 8; p++) lds_dma16s(src + p * 2 * kHeadDim, cb ^ ((uint32_t)p << jsh), lds + p * 1024);
    };
    const uint32_t ku = lds_addr(&sm.unit[2 * wave][0]), vu = ku + kUnitLds;
    if (n_my > 0) {
        issue(a.kpool, cbk, 5, 0, ku);
        issue(a.vpool, cbv, 6, 0, vu);
    }

    f32x4 o[T][16];
    float m_run[T], l[T];  // l: the lane's part of the row's sum of weights
#pragma unroll
    for (int t = 0; t < T; t++) {
        m_run[t] = kNegBig;
        l[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < 16; dt++) o[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // operand fragments within a unit: K (ks = 4 hi + jj): (ka ^ 64 jj) + 256 hi;
    // V^T (dt): va ^ 32 dt; the swizzles are in ka and va
    const int vr = 4 * q4 + (r16 >> 2);  // V row % 16 of this lane
    uint32_t ka = ku + r16 * 512 + 16 * (q4 ^ r16);
    uint32_t va = vu + vr * (512 + 32) + 8 * (r16 & 3);

    for (int i = 0; i < n_my; i++) {
        const bool more = i + 1 < n_my;
        asm volatile("" : "+v"(ka), "+v"(va));  // (the fragments' addresses are not kept over the loop)
        wait_vm<8>();  // K: the 8 copies after it are V's
        f32x4 st[T];
        {
            bf16x8_t kf[kShAhead];
            auto read = [&](int ks) {
                kf[ks % kShAhead] = as_bf16x8(lds_load16(ka ^ (64 * (ks & 3)), 256 * (ks >> 2)));
            };
#pragma unroll
            for (int n = 0; n < kShAhead; n++) read(n);
#pragma unroll
            for (int ks = 0; ks < 8; ks++) {
                const bf16x8_t x = kf[ks % kShAhead];
                if (ks + kShAhead < 8) read(ks + kShAhead);
#pragma unroll
                for (int t = 0; t < T; t++)
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, qb[t][ks], ks == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : st[t], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_group_barrier(kSgDsRead, kShAhead, 0);
#pragma unroll
        for (int n = 0; n < 8; n++) {
            if (n + kShAhead < 8) __builtin_amdgcn_sched_group_barrier(kSgDsRead, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kSgMfma, T, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        wait_lds();
        if (more) issue(a.kpool, cbk, 5, i + 1, ku);
        // weights of the scores
        bf16x4_t pw[T][PARTS];
#pragma unroll
        for (int t = 0; t < T; t++) {
            const float mx = fmaxf(fmaxf(st[t][0], st[t][1]), fmaxf(st[t][2], st[t][3]));
            const float mt = max_xor32(max_xor16(mx)) * c;
            const bool up = mt > m_run[t] + kRescaleSlack;
            if (__builtin_amdgcn_ballot_w64(up) != 0) {  // uniform; rows that keep their maximum scale by 1
                const float cr = up ? fast_exp2(m_run[t] - mt) : 1.f;
                m_run[t] = up ? mt : m_run[t];
#pragma unroll
                for (int dt = 0; dt < 16; dt++) o[t][dt] *= cr;
                l[t] *= cr;
            }
            const float nm = -m_run[t];
            u32x2 w[PARTS];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float x = fast_exp2(fmaf(st[t][2 * e], c, nm)), y = fast_exp2(fmaf(st[t][2 * e + 1], c, nm));
                w[0][e] = cvt_pk_bf16(x, y);
                if constexpr (PARTS == 1) {
                    l[t] += bf16lo(w[0][e]) + bf16hi(w[0][e]);  // what the product uses
                } else {
                    l[t] += x + y;
                    const float x1 = x - bf16lo(w[0][e]), y1 = y - bf16hi(w[0][e]);  // exact
                    w[1][e] = cvt_pk_bf16(x1, y1);
                    w[2][e] = cvt_pk_bf16(x1 - bf16lo(w[1][e]), y1 - bf16hi(w[1][e]));
                }
            }
#pragma unroll
            for (int p = 0; p < PARTS; p++) pw[t][p] = __builtin_bit_cast(bf16x4_t, w[p]);
        }
        if (more)
            wait_vm<8>();
        else
            wait_vm<0>();
        {
            bf16x4_t vf[kShAhead];
            auto read = [&](int dt) { vf[dt % kShAhead] = __builtin_bit_cast(bf16x4_t, lds_load_tr16(va ^ (32 * dt), 0)); };
#pragma unroll
            for (int n = 0; n < kShAhead; n++) read(n);
#pragma unroll
            for (int dt = 0; dt < 16; dt++) {
                const bf16x4_t x = vf[dt % kShAhead];
                if (dt + kShAhead < 16) read(dt + kShAhead);
#pragma unroll
                for (int t = 0; t < T; t++)
#pragma unroll
                    for (int p = 0; p < PARTS; p++)
                        o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(x, pw[t][p], o[t][dt], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_group_barrier(kSgDsRead, kShAhead, 1);
#pragma unroll
        for (int n = 0; n < 16; n++) {
            if (n + kShAhead < 16) __builtin_amdgcn_sched_group_barrier(kSgDsRead, 1, 1);
            __builtin_amdgcn_sched_group_barrier(kSgMfma, T * PARTS, 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        wait_lds();
        if (more) issue(a.vpool, cbv, 6, i + 1, vu);
    }
    int row[T];  // of the lane's partial
#pragma unroll
    for (int t = 0; t < T; t++) {
        l[t] = sum_xor32(sum_xor16(l[t]));
        const int e = entry(t), r0 = __builtin_amdgcn_ds_bpermute((e & 63) * 4, seq_row);  // lane s holds sequence s's
        row[t] = (r0 + (e >> 6) + it.ck) * kQHeads + h * kGroup + g;
    }

    if (it.kind == kSharedHeads) {
#pragma unroll
        for (int t = 0; t < T; t++) {
            if (4 * t + (r16 >> 2) >= it.members) continue;
            float* acc = a.acc + (size_t)row[t] * kHeadDim + 4 * q4;
#pragma unroll
            for (int dt = 0; dt < 16; dt++) *reinterpret_cast<f32x4*>(acc + 16 * dt) = o[t][dt];
            if (q4 == 0) *reinterpret_cast<float2*>(a.stats + (size_t)row[t] * 2) = make_float2(m_run[t], l[t]);
        }
        return;
    }
    // fold the 4 waves' keys, tile by tile: O through LDS (each wave into its own
    // units, which it alone read), 16-B chunks swizzled by the row; then a wave takes
    // a member
    uint8_t* own = reinterpret_cast<uint8_t*>(sm.unit[2 * wave]);
#pragma unroll
    for (int t = 0; t < T; t++) {
        if (t > 0) __syncthreads();
#pragma unroll
        for (int dt = 0; dt < 16; dt++)
            *reinterpret_cast<f32x4*>(own + r16 * 1024 + (((4 * dt + q4) ^ r16) << 4)) = o[t][dt];
        if (q4 == 0) sm.ml[wave][r16] = make_float2(m_run[t], l[t]);
        __syncthreads();
        if (4 * t + wave >= it.members) continue;  // uniform
#pragma unroll
        for (int rr = 0; rr < kGroup; rr++) {
            const int r = kGroup * wave + rr;
            float2 ml[kWaves];
            f32x4 x[kWaves];
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                ml[w] = sm.ml[w][r];
                x[w] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const uint8_t*>(sm.unit[2 * w]) + r * 1024 + ((lane ^ r) << 4));
            }
            const float m = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
            float lt = 0.f;
            f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                const float f = fast_exp2(ml[w].x - m);
                lt = fmaf(f, ml[w].y, lt);
                y += f * x[w];
            }
            const size_t to = (size_t)__builtin_amdgcn_readlane(row[t], r);  // lane r holds row r's
            *reinterpret_cast<f32x4*>(a.acc + to * kHeadDim + lane * 4) = y;
            if (lane == 0) *reinterpret_cast<float2*>(a.stats + to * 2) = make_float2(m, lt);
        }
    }
}

// A chunk of one sequence: 4 rows, read from memory once.  The walk of
// kvc_decode_attn holds twice the bytes in flight that the tiles' LDS does.
template <int PARTS>
__device__ __forceinline__ void shared_one(const SharedArgs& a, const SharedItem& it, int seq_row, SharedOneSmem& sm) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n_blk = (it.keys + kBlockTok - 1) / kBlockTok, e = it.who[0] & 0xFFFF;
    const int ids = lane < min(64, n_blk) ? it.trow[lane] : 0;
    __builtin_amdgcn_sched_barrier(0);
    uint32_t qv[kGroup][2][4];
    load_q(qv, a.q + ((size_t)(e & 63) * kQHeads + it.h * kGroup) * kHeadDim, lane);
    WaveState st;
    init_state(st);
    walk_blocks<1, false, PARTS != 1>(a.kpool, a.vpool, it.trow, it.h, 0, n_blk, it.keys, qv, a.scale_log2,
                                      reinterpret_cast<uint16_t*>(sm.p[wave]), st, wave, lane, 0, ids, [] {});
    finalize_l(st);
    float m, l, A[4];
    merge_waves(st, sm.d, wave, lane, m, l, A);  // head `wave`, dims 4 lane ..
    const size_t row = (size_t)(__builtin_amdgcn_readlane(seq_row, e & 63) + (e >> 6) + it.ck) * kQHeads + it.h * kGroup + wave;
    *reinterpret_cast<float4*>(a.acc + row * kHeadDim + lane * 4) = make_float4(A[0], A[1], A[2], A[3]);
    if (lane == 0) *reinterpret_cast<float2*>(a.stats + row * 2) = make_float2(m, l);
}

// (2 waves a SIMD: two workgroups on a CU, up to 256 registers a wave)
template <int PARTS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void shared_decode_kernel(SharedArgs a) {
    __shared__ __align__(1024) union {  // (the XORs with a fragment's number need it)
        SharedSmem tiles;
        SharedOneSmem one;
    } sm;
    const int lane = threadIdx.x & 63;
    const int item = blockIdx.x;
    // one trip to the arguments: every lane asks for the ends and records of two
    // nodes, 8 list entries and a sequence's first partial
    int e0 = a.item_end[lane], e1 = a.item_end[lane + 64];
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    i32x4 n0 = *reinterpret_cast<const i32x4*>(&a.node[lane]), n1 = *reinterpret_cast<const i32x4*>(&a.node[lane + 64]);
    i32x4 mw = *reinterpret_cast<const i32x4*>(&a.member[8 * lane]);
    int seq_row = a.seq_row[lane];
    asm volatile("" : "+v"(e0), "+v"(e1), "+v"(n0), "+v"(n1), "+v"(mw), "+v"(seq_row));  // all of it, here
    const int node = __popcll(__builtin_amdgcn_ballot_w64(e0 <= item)) + __popcll(__builtin_amdgcn_ballot_w64(e1 <= item));
    if (node >= kSharedNodes) return;
    const int at = node & 63;
    const bool up = node >= 64;
    const uint32_t w0 = up ? __builtin_amdgcn_readlane(n1.x, at) : __builtin_amdgcn_readlane(n0.x, at);
    const uint32_t w1 = up ? __builtin_amdgcn_readlane(n1.y, at) : __builtin_amdgcn_readlane(n0.y, at);
    const uint32_t w2 = up ? __builtin_amdgcn_readlane(n1.z, at) : __builtin_amdgcn_readlane(n0.z, at);
    const int slot = up ? __builtin_amdgcn_readlane(n1.w, at) : __builtin_amdgcn_readlane(n0.w, at);
    const int begin = node == 0 ? 0 : node <= 64 ? __builtin_amdgcn_readlane(e0, node - 1) : __builtin_amdgcn_readlane(e1, node - 65);
    constexpr uint32_t kLow26 = (1u << 26) - 1;
    const int first = w0 & kLow26, len = w1 & kLow26, chunk = w2 & 1023;
    if (len == 0) return;  // (behind the last node)
    const int all = (w2 >> 10 & 63) + 1;  // members of the node
    SharedItem it;
    it.kind = w0 >> 26;
    const int n_chunks = (len + chunk - 1) / chunk, units = it.kind == kSharedHeads ? n_chunks : n_chunks * kKvHeads;
    const int size = all > 1 && (w2 >> 22 & 1) ? kSharedTile : kSharedSeqs;  // of a group
    int j = item - begin, grp = 0;
    if (all > size) {
        // (the node starts on a multiple of 8; the groups of members that read the
        // same keys run on one XCD, workgroup number % 8, one after the other)
        const int groups = (all + size - 1) / size;
        j = item - (begin + 7) / 8 * 8;
        if (j < 0) return;
        const int r = j >> 3;
        grp = r % groups;
        j = r / groups * 8 + (j & 7);
    }
    if (j >= units) return;  // (padding)
    it.h = it.kind == kSharedHeads ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : j % kKvHeads;
    it.ck = it.kind == kSharedHeads ? j : j / kKvHeads;
    const int b0 = it.ck * chunk;
    const int n_blk = min(chunk, len - b0);
    it.keys = n_blk * kBlockTok - (b0 + n_blk == len ? kBlockTok - 1 - (int)(w1 >> 26) : 0);
    it.members = min(size, all - grp * size);
    it.trow = a.table + (size_t)slot * a.table_stride + first + b0;
    if (all == 1) {
        it.who[0] = it.who[1] = it.who[2] = it.who[3] = (w2 >> 16) * 0x10001u;
    } else {
        const int from = (w2 >> 16 & 63) + grp * size / 8;  // lane that holds them
        it.who[0] = __builtin_amdgcn_readlane(mw.x, from);
        it.who[1] = __builtin_amdgcn_readlane(mw.y, from);
        it.who[2] = __builtin_amdgcn_readlane(mw.z, from);
        it.who[3] = __builtin_amdgcn_readlane(mw.w, from);
        if (size == kSharedTile && (grp & 1)) {  // the list's second half
            it.who[0] = it.who[2];
            it.who[1] = it.who[3];
        }
    }
    if (it.kind == kSharedOne)
        shared_one<PARTS>(a, it, seq_row, sm.one);
    else if (it.members > 4)
        shared_item<2, PARTS>(a, it, seq_row, sm.tiles);
    else
        shared_item<1, PARTS>(a, it, seq_row, sm.tiles);
}

// One workgroup folds a (sequence, q head): each wave every 4th partial, its
// first kSharedFold requested before the weights are known.  The new token is
// a partial of its own, (score, 1, v), and is written to the cache.
constexpr int kSharedFold = 16;
constexpr int kSharedFew = 16;
__global__ __launch_bounds__(256) void shared_fold_kernel(SharedFoldArgs a) {
    __shared__ float wgt[kSharedPath];
    __shared__ float red[kWaves][2];
    __shared__ f32x4 part[kWaves][64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int s = blockIdx.x / kQHeads, head = blockIdx.x % kQHeads, h = head / kGroup, g = head % kGroup;
    const SharedSeq sq = a.seq[s];
    const int np = sq.parts;
    const size_t row0 = (size_t)sq.row * kQHeads + head;
    const size_t qrow = ((size_t)s * kQHeads + head) * kHeadDim;
    const bool has_gate = a.gate != nullptr;
    uint2 gw = make_uint2(0u, 0u);
    if (has_gate) gw = *reinterpret_cast<const uint2*>(a.gate + qrow + lane * 4);
    uint2 qw = make_uint2(0u, 0u), kw = qw, vw = qw;
    if (a.k_new) {
        const size_t krow = ((size_t)s * kKvHeads + h) * kHeadDim + lane * 4;
        qw = *reinterpret_cast<const uint2*>(a.q + qrow + lane * 4);
        kw = *reinterpret_cast<const uint2*>(a.k_new + krow);
        vw = *reinterpret_cast<const uint2*>(a.v_new + krow);
    }
    f32x4 x[kSharedFold];
    if (np > 0) {
#pragma unroll
        for (int k = 0; k < kSharedFold; k++)
            x[k] = *reinterpret_cast<const f32x4*>(a.acc + (row0 + (size_t)min(wave + kWaves * k, np - 1) * kQHeads) * kHeadDim + lane * 4);
    }
    float ms[kSharedPath / 256], ls[kSharedPath / 256], m = kNegBig;
#pragma unroll
    for (int i = 0; i < kSharedPath / 256; i++) {
        ms[i] = kNegBig;
        ls[i] = 0.f;
        if (tid + 256 * i < np) {
            const float2 t = *reinterpret_cast<const float2*>(a.stats + (row0 + (size_t)(tid + 256 * i) * kQHeads) * 2);
            ms[i] = t.x;
            ls[i] = t.y;
        }
        m = fmaxf(m, ms[i]);
    }
    float sc = kNegBig;
    if (a.k_new) {
        sc = wave_sum(bf16lo(qw.x) * bf16lo(kw.x) + bf16hi(qw.x) * bf16hi(kw.x) + bf16lo(qw.y) * bf16lo(kw.y) +
                      bf16hi(qw.y) * bf16hi(kw.y)) * a.scale_log2;
        m = fmaxf(m, sc);
    }
    m = wave_max(m);
    if (lane == 0) red[wave][0] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < kSharedPath / 256; i++) {
        const float f = fast_exp2(ms[i] - m);
        if (tid + 256 * i < np) wgt[tid + 256 * i] = f;
        l = fmaf(f, ls[i], l);
    }
    l = wave_sum(l);
    if (lane == 0) red[wave][1] = l;
    __syncthreads();
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kSharedFold; k++)
        if (wave + kWaves * k < np) t += wgt[wave + kWaves * k] * x[k];
    for (int p = wave + kWaves * kSharedFold; p < np; p += kWaves)
        t += wgt[p] * *reinterpret_cast<const f32x4*>(a.acc + (row0 + (size_t)p * kQHeads) * kHeadDim + lane * 4);
    part[wave][lane] = t;
    __syncthreads();
    if (wave != 0) return;
    l = red[0][1] + red[1][1] + red[2][1] + red[3][1];
    t = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
    float A[4] = {t[0], t[1], t[2], t[3]};
    if (a.k_new) {
        const float f = fast_exp2(sc - m);
        l += f;
        A[0] = fmaf(f, bf16lo(vw.x), A[0]);
        A[1] = fmaf(f, bf16hi(vw.x), A[1]);
        A[2] = fmaf(f, bf16lo(vw.y), A[2]);
        A[3] = fmaf(f, bf16hi(vw.y), A[3]);
        if (g == 0) {
            const int pos = sq.keys;
            const int blk = a.table[(size_t)sq.slot * a.table_stride + pos / kBlockTok];
            const size_t off = (((size_t)blk * kKvHeads + h) * kBlockTok + pos % kBlockTok) * kHeadDim + lane * 4;
            *reinterpret_cast<uint2*>(a.kpool + off) = kw;
            *reinterpret_cast<uint2*>(a.vpool + off) = vw;
        }
    }
    float gs[4] = {1.f, 1.f, 1.f, 1.f};
    if (has_gate) gate_factors(gw, a.gate_ref, gs);
    write_out(a.out, a.out_bf16, qrow, lane * 4, has_gate, gs, l, A);
}

// The same for few partials: a wave folds a q head alone, a workgroup a kv head.
__global__ __launch_bounds__(256) void shared_fold_few_kernel(SharedFoldArgs a) {
    const int lane = threadIdx.x & 63, g = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int s = blockIdx.x / kKvHeads, h = blockIdx.x % kKvHeads, head = h * kGroup + g;
    const SharedSeq sq = a.seq[s];
    const int np = sq.parts;
    const size_t row0 = (size_t)sq.row * kQHeads + head;
    const size_t qrow = ((size_t)s * kQHeads + head) * kHeadDim;
    const bool has_gate = a.gate != nullptr;
    uint2 gw = make_uint2(0u, 0u), qw = gw, kw = gw, vw = gw;
    if (has_gate) gw = *reinterpret_cast<const uint2*>(a.gate + qrow + lane * 4);
    int blk = 0;
    if (a.k_new) {
        const size_t krow = ((size_t)s * kKvHeads + h) * kHeadDim + lane * 4;
        qw = *reinterpret_cast<const uint2*>(a.q + qrow + lane * 4);
        kw = *reinterpret_cast<const uint2*>(a.k_new + krow);
        vw = *reinterpret_cast<const uint2*>(a.v_new + krow);
        if (g == 0) blk = a.table[(size_t)sq.slot * a.table_stride + sq.keys / kBlockTok];
    }
    float2 ml = make_float2(kNegBig, 0.f);
    f32x4 x[kSharedFew];
    if (np > 0) {
        if (lane < np) ml = *reinterpret_cast<const float2*>(a.stats + (row0 + (size_t)lane * kQHeads) * 2);
#pragma unroll
        for (int k = 0; k < kSharedFew; k++)
            x[k] = *reinterpret_cast<const f32x4*>(a.acc + (row0 + (size_t)min(k, np - 1) * kQHeads) * kHeadDim + lane * 4);
    }
    float m = wave_max(ml.x), sc = kNegBig;
    if (a.k_new) {
        sc = wave_sum(bf16lo(qw.x) * bf16lo(kw.x) + bf16hi(qw.x) * bf16hi(kw.x) + bf16lo(qw.y) * bf16lo(kw.y) +
                      bf16hi(qw.y) * bf16hi(kw.y)) * a.scale_log2;
        m = fmaxf(m, sc);
    }
    const float f = lane < np ? fast_exp2(ml.x - m) : 0.f;
    float l = wave_sum(f * ml.y);
    float A[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kSharedFew; k++) {
        if (k < np) {  // uniform
            const float w = readlane(f, k);
#pragma unroll
            for (int i = 0; i < 4; i++) A[i] = fmaf(w, x[k][i], A[i]);
        }
    }
    if (a.k_new) {
        const float w = fast_exp2(sc - m);
        l += w;
        A[0] = fmaf(w, bf16lo(vw.x), A[0]);
        A[1] = fmaf(w, bf16hi(vw.x), A[1]);
        A[2] = fmaf(w, bf16lo(vw.y), A[2]);
        A[3] = fmaf(w, bf16hi(vw.y), A[3]);
        if (g == 0) {
            const size_t off = (((size_t)blk * kKvHeads + h) * kBlockTok + sq.keys % kBlockTok) * kHeadDim + lane * 4;
            *reinterpret_cast<uint2*>(a.kpool + off) = kw;
            *reinterpret_cast<uint2*>(a.vpool + off) = vw;
        }
    }
    float gs[4] = {1.f, 1.f, 1.f, 1.f};
    if (has_gate) gate_factors(gw, a.gate_ref, gs);
    write_out(a.out, a.out_bf16, qrow, lane * 4, has_gate, gs, l, A);
}

int launch_shared(const SharedArgs& a, int32_t n_items, const SharedFoldArgs& f, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    if (n_items > 0) {
        if (f.out_bf16)
            hipLaunchKernelGGL(shared_decode_kernel<1>, dim3(n_items), dim3(kWaves * 64), 0, st, a);
        else
            hipLaunchKernelGGL(shared_decode_kernel<3>, dim3(n_items), dim3(kWaves * 64), 0, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    int32_t parts = 0;
    for (int32_t i = 0; i < f.n_seqs; i++) parts = f.seq[i].parts > parts ? f.seq[i].parts : parts;
    if (parts <= kSharedFew)
        hipLaunchKernelGGL(shared_fold_few_kernel, dim3(f.n_seqs * kKvHeads), dim3(256), 0, st, f);
    else
        hipLaunchKernelGGL(shared_fold_kernel, dim3(f.n_seqs * kQHeads), dim3(256), 0, st, f);
    return (int)hipGetLastError();
}

}  // namespace kvc
