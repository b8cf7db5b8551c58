// kvc_evict_kernels.h -- kernels of eviction by accumulated attention weight:
// the weights that query rows give every cached token, the choice of the
// tokens that stay, and the move of their rows.  Included by kvc_kernels.hip.
#pragma once

namespace kvc {

// ---------------------------------------------------------------------------
// Attention weights: acc[key] += sum over rows of 2^(s - m_row) / l_row, with
// s the row's score in the log2 domain, m_row and l_row its maximum and sum
// over every key.  No weight is known before the last key's score is, so the
// keys are passed twice, in two launches.
//
// A wave takes one block of one kv head.  The block's K sits in registers as A
// operand (keys x dims; 8-bit blocks as exact bf16 integers, scaled after the
// product), and the rows (row 4 i + g = query i, q head g of the group) pass
// by in tiles of 16 as B operand, 128 rows at a time out of LDS, where they lie
// in operand order for all 8 waves.  (Read from memory by every wave, 64 KB of
// rows beside 8 of keys, they took the L1 path 3 times as long: 16 sequences x
// 32 queries 119 us, with LDS 51.)  A lane then has 8 keys of one row.
//
// Few rows are bound by memory, or by two launches' latency: 64 sequences of
// 500..8000 tokens, 1 query, bf16 124 + 22 us, 4.0 TB/s; 1 x 4096 10 us (6 and 4).
// In 8 bits the 64 sequences take 82 + 22 us, 2.9 TB/s: a wave has one block to
// ask for and to widen, and waits 59 % of its cycles.  Many rows wait too: 16 x 32
// queries over 500..6000 8-bit tokens 25 and 27 us, each 11.8 GFLOP and 52 MB;
// the matrix pipe is busy 20-22 % of the cycles, VALU 31-34 % (exponentials
// counted as any other instruction), LDS 13-17 %, and the waves spend 48 % of
// theirs at waits (each workgroup's rows and keys, once, with nothing beside).
__device__ __forceinline__ void weights_load_k(u32x4 (&kf)[2][8], const MixedCache& c, int id, int h, bool q8, int lane) {
    const int r16 = lane & 15, g = lane >> 4;
    const size_t unit = (size_t)id * kKvHeads + h;
    if (q8) {
        // piece (t, s, 16 g' + c) holds dims 64 s + 16 g' ..: operand slice
        // 2 s + half takes dims 64 s + 32 half + 8 g .., half a piece
        const uint8_t* k = c.k8 + unit * kQ8UnitBytes;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int ks = 0; ks < 8; ks++) {
                const int gp = 2 * (ks & 1) + (g >> 1);
                const u32x2 w = *reinterpret_cast<const u32x2*>(
                    k + (((t * 4 + (ks >> 1)) * 64 + 16 * gp + r16) * 16 + 8 * (g & 1)));
                const u32x2 lo = i8x4_to_bf16(w[0]), hi = i8x4_to_bf16(w[1]);
                kf[t][ks] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            }
    } else {
        const uint16_t* k = c.kpool + unit * kBlockTok * kHeadDim;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int ks = 0; ks < 8; ks++)
                kf[t][ks] = *reinterpret_cast<const u32x4*>(k + (16 * t + r16) * kHeadDim + 32 * ks + 8 * g);
    }
}

// Bytes from the sequence's first query to the lane's piece of B operand slice
// ks (dims 32 ks + 8 (lane / 16) ..) of row r0 + lane % 16; rows past the last
// repeat it.
__device__ __forceinline__ uint32_t weights_q(const WeightsArgs& a, int h, int r0, int ks, int lane) {
    const int rc = min(r0 + (lane & 15), a.n_q * kGroup - 1);
    return (((rc >> 2) * kQHeads + h * kGroup + (rc & 3)) * kHeadDim + 32 * ks + 8 * (lane >> 4)) * 2;
}

// Rows g0 .. end - 1 into LDS as [tile][ks][lane], the waves in turn a slice.
__device__ __forceinline__ void weights_stage_q(uint32_t lds, const WeightsArgs& a, const uint16_t* q, int h, int g0, int end,
                                                int wave, int waves, int lane) {
    for (int i = wave; i < ((end - g0 + 15) >> 4) * 8; i += waves)
        lds_dma16s(q, weights_q(a, h, g0 + 16 * (i >> 3), i & 7, lane), lds + i * 1024);
}

// Raw products of the lane's keys 16 t + 4 (lane / 16) + i with one row.
__device__ __forceinline__ void weights_product(f32x4 (&st)[2], const u32x4 (&kf)[2][8], const u32x4 (&qf)[8]) {
#pragma unroll
    for (int t = 0; t < 2; t++) st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 8; ks++)
#pragma unroll
        for (int t = 0; t < 2; t++)
            st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kf[t][ks]), as_bf16x8(qf[ks]), st[t], 0, 0, 0);
}

// -infinity for the keys from key0 on that row r0 + lane % 16 does not see.
__device__ __forceinline__ void weights_mask(f32x4 (&st)[2], const WeightsArgs& a, int L, int key0, int r0, int lane) {
    const int last = L - a.n_q + (min(r0 + (lane & 15), a.n_q * kGroup - 1) >> 2) - key0;  // last one it sees
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (16 * t + 4 * (lane >> 4) + i > last) st[t][i] = -__builtin_inff();
}

// First launch: (max, sum 2^(s - max)) of every row over a chunk of a.chunk
// blocks.  STORE: one tile of rows, whose scores go to the workspace, one block
// per wave; otherwise the waves share the chunk's blocks, and those of a block
// its tiles.
template <bool STORE>
__global__ __launch_bounds__(64 * weights_waves(STORE), 4) void weights_score_kernel(WeightsArgs a) {
    constexpr int W = weights_waves(STORE), ROWS = STORE ? 16 : kWeightsRows;
    __shared__ float2 ml[W][ROWS];
    __shared__ u32x4 qs[STORE ? 1 : ROWS * kHeadDim / 8];
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunk = blockIdx.x >> 2, h = blockIdx.x & 3;
    const int s = find_seq(a.chunk_begin, a.n_seqs, chunk);
    const int L = a.kv_len[s], R = a.n_q * kGroup;
    const int nb = (L + kBlockTok - 1) / kBlockTok;
    const int bw = STORE ? wave : wave & (a.chunk - 1);  // its block of the chunk
    const int b = (chunk - a.chunk_begin[s]) * a.chunk + bw;
    const int tile0 = STORE ? 0 : 16 * wave / a.chunk & ~15, tiles = STORE ? 16 : 16 * W / a.chunk;
    const bool masked = (b + 1) * kBlockTok > L - a.n_q + 1;  // a key that some row does not see
    const uint16_t* q = a.q + (size_t)s * a.n_q * kQHeads * kHeadDim;
    u32x4 kf[2][8];
    float scale = a.scale_log2;
    if (!STORE) weights_stage_q(lds_addr(qs), a, q, h, 0, min(ROWS, R), wave, W, lane);
    if (b < nb) {
        const int id = a.c.table[(size_t)a.slot[s] * a.c.table_stride + b];
        const bool q8 = b < a.n8[s];
        weights_load_k(kf, a.c, id, h, q8, lane);
        if (q8) scale *= a.c.ks[(size_t)id * kKvHeads + h];
    }
    float2* stats = reinterpret_cast<float2*>(a.stats) + ((size_t)h * a.total_chunks + chunk) * R;
    for (int g0 = 0; g0 < R; g0 += ROWS) {
        const int end = min(g0 + ROWS, R);
        if (!STORE) {
            if (g0) weights_stage_q(lds_addr(qs), a, q, h, g0, end, wave, W, lane);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
        if (b < nb) {
            for (int r0 = g0 + tile0; r0 < end; r0 += tiles) {
                u32x4 qf[8];
#pragma unroll
                for (int ks = 0; ks < 8; ks++)
                    qf[ks] = STORE ? *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(q) + weights_q(a, h, r0, ks, lane))
                                   : qs[((r0 - g0) / 2 + ks) * 64 + lane];
                f32x4 st[2];
                weights_product(st, kf, qf);
#pragma unroll
                for (int t = 0; t < 2; t++) st[t] *= scale;
                if (masked) weights_mask(st, a, L, b * kBlockTok, r0, lane);
                float mx = kNegBig;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) mx = fmaxf(mx, st[t][i]);
                mx = max_xor16(mx);
                mx = max_xor32(mx);
                float l = 0.f;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) l += fast_exp2(st[t][i] - mx);  // 0 for -infinity
                l = sum_xor16(l);
                l = sum_xor32(l);
                if (STORE && r16 < R) {
                    float* out = a.scores + (((size_t)h * a.total_blocks + a.block_begin[s] + b) * R + r16) * kBlockTok;
#pragma unroll
                    for (int t = 0; t < 2; t++) *reinterpret_cast<f32x4*>(out + 16 * t + 4 * g) = st[t];
                }
                if (g == 0) ml[bw][r0 - g0 + r16] = make_float2(mx, l);
            }
        } else {
            for (int r = lane; r < ROWS; r += 64) ml[bw][r] = make_float2(kNegBig, 0.f);
        }
        __syncthreads();
        for (int r = threadIdx.x; r < end - g0; r += 64 * W) {
            float m = kNegBig, l = 0.f;
            for (int w = 0; w < a.chunk; w++) m = fmaxf(m, ml[w][r].x);
            for (int w = 0; w < a.chunk; w++) l = fmaf(fast_exp2(ml[w][r].x - m), ml[w][r].y, l);
            stats[g0 + r] = make_float2(m, l);
        }
        __syncthreads();
    }
}

// Folds (max, sum) of two parts of a row.
__device__ __forceinline__ float2 weights_fold(float2 x, float2 y) {
    const float m = fmaxf(x.x, y.x);
    return make_float2(m, fmaf(x.y, fast_exp2(x.x - m), y.y * fast_exp2(y.x - m)));
}

// (max, 1 / sum) of the R <= 16 rows over the nc chunks of a sequence: LANES
// neighbouring threads of 256 share a row and take every LANES'th chunk of it.
__device__ __forceinline__ void weights_few_rows(float2* row_ml, const float2* stats, int R, int nc, int t) {
    int lanes = 64;
    while (lanes * R > 256) lanes >>= 1;
    const int r = t / lanes;
    float2 x = make_float2(kNegBig, 0.f);
    if (r < R)
#pragma unroll 4
        for (int k = t % lanes; k < nc; k += lanes) x = weights_fold(x, stats[(size_t)k * R + r]);
    for (int d = lanes >> 1; d > 0; d >>= 1) x = weights_fold(x, make_float2(__shfl_xor(x.x, d), __shfl_xor(x.y, d)));
    if (t % lanes == 0 && r < R) row_ml[r] = make_float2(x.x, 1.0f / x.y);
}

// The same of n <= kWeightsRows rows from g0 on: neighbouring threads take
// neighbouring rows, each of the PARTS groups of threads every PARTS'th chunk.
// Rows from n on count for nothing: 2^(s - inf).
template <int THREADS>
__device__ __forceinline__ void weights_rows(float2* row_ml, float2* part, const float2* stats, int R, int g0, int n, int nc, int t) {
    const int wide = n > 64 ? 128 : n > 32 ? 64 : 32, parts = THREADS / wide;
    const int r = t % wide;
    float2 x = make_float2(kNegBig, 0.f);
    if (r < n)
#pragma unroll 4
        for (int k = t / wide; k < nc; k += parts) x = weights_fold(x, stats[(size_t)k * R + g0 + r]);
    part[t] = x;
    __syncthreads();
    if (t < kWeightsRows) {
        if (t < n)
            for (int k = 1; k < parts; k++) x = weights_fold(x, part[k * wide + t]);
        row_ml[t] = t < n ? make_float2(x.x, 1.0f / x.y) : make_float2(__builtin_inff(), 0.f);
    }
}

// Second launch after stored scores: one workgroup = kWsumBlocks blocks of one
// kv head; thread (key, block) sums its key's weights over the rows in order
// and adds them to the accumulator: no atomics, the same bits each time.
__global__ __launch_bounds__(256) void weights_sum_kernel(WeightsArgs a) {
    __shared__ float2 row_ml[16];
    const int t = threadIdx.x;
    const int item = blockIdx.x >> 2, h = blockIdx.x & 3;
    const int s = find_seq(a.sum_begin, a.n_seqs, item);
    const int L = a.kv_len[s], R = a.n_q * kGroup;
    const int nb = (L + kBlockTok - 1) / kBlockTok;
    const int b = (item - a.sum_begin[s]) * kWsumBlocks + (t >> 5), key = t & 31;
    const int pos = b * kBlockTok + key;
    const bool in = b < nb && pos < L;
    const size_t o = ((size_t)s * kKvHeads + h) * (size_t)a.stride + pos;
    const float* sc = a.scores + ((size_t)h * a.total_blocks + a.block_begin[s] + b) * R * kBlockTok + key;
    // asked for before the statistics are folded
    const float before = in && a.acc_in ? a.acc_in[o] : 0.f;
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; r++) x[r] = in && r < R ? sc[(size_t)r * kBlockTok] : 0.f;
    weights_few_rows(row_ml, reinterpret_cast<const float2*>(a.stats) + ((size_t)h * a.total_chunks + a.chunk_begin[s]) * R,
                     R, a.chunk_begin[s + 1] - a.chunk_begin[s], t);
    __syncthreads();
    if (!in) return;
    float w = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r++)
        if (r < R) w = fmaf(fast_exp2(x[r] - row_ml[r].x), row_ml[r].y, w);
    a.acc_out[o] = before + w;
}

// Second launch without stored scores: the same waves compute them again.  A
// lane sums its 8 keys' weights over the tiles in order; the 16 lanes of a key
// and then the waves of a block are added at the end: the same bits each time.
__global__ __launch_bounds__(64 * weights_waves(false), 4) void weights_again_kernel(WeightsArgs a) {
    constexpr int W = weights_waves(false), ROWS = kWeightsRows;
    __shared__ float2 row_ml[ROWS];
    __shared__ float2 part[64 * W];
    __shared__ float sums[W][kBlockTok];
    __shared__ u32x4 qs[ROWS * kHeadDim / 8];
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunk = blockIdx.x >> 2, h = blockIdx.x & 3;
    const int s = find_seq(a.chunk_begin, a.n_seqs, chunk);
    const int L = a.kv_len[s], R = a.n_q * kGroup;
    const int nb = (L + kBlockTok - 1) / kBlockTok;
    const int b = (chunk - a.chunk_begin[s]) * a.chunk + (wave & (a.chunk - 1));
    const int tile0 = 16 * wave / a.chunk & ~15, tiles = 16 * W / a.chunk;
    const bool masked = (b + 1) * kBlockTok > L - a.n_q + 1;
    const uint16_t* q = a.q + (size_t)s * a.n_q * kQHeads * kHeadDim;
    u32x4 kf[2][8];
    float scale = a.scale_log2;
    weights_stage_q(lds_addr(qs), a, q, h, 0, min(ROWS, R), wave, W, lane);
    if (b < nb) {
        const int id = a.c.table[(size_t)a.slot[s] * a.c.table_stride + b];
        const bool q8 = b < a.n8[s];
        weights_load_k(kf, a.c, id, h, q8, lane);
        if (q8) scale *= a.c.ks[(size_t)id * kKvHeads + h];
    }
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + ((size_t)h * a.total_chunks + a.chunk_begin[s]) * R;
    const int nc = a.chunk_begin[s + 1] - a.chunk_begin[s];
    f32x4 w[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    for (int g0 = 0; g0 < R; g0 += ROWS) {
        const int end = min(g0 + ROWS, R);
        if (g0) {
            __syncthreads();
            weights_stage_q(lds_addr(qs), a, q, h, g0, end, wave, W, lane);
        }
        weights_rows<64 * W>(row_ml, part, stats, R, g0, end - g0, nc, threadIdx.x);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (b >= nb) continue;
        for (int r0 = g0 + tile0; r0 < end; r0 += tiles) {
            u32x4 qf[8];
#pragma unroll
            for (int ks = 0; ks < 8; ks++) qf[ks] = qs[((r0 - g0) / 2 + ks) * 64 + lane];
            const float2 x = row_ml[r0 - g0 + r16];
            f32x4 st[2];
            weights_product(st, kf, qf);
#pragma unroll
            for (int t = 0; t < 2; t++) st[t] *= scale;
            if (masked) weights_mask(st, a, L, b * kBlockTok, r0, lane);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) w[t][i] = fmaf(fast_exp2(st[t][i] - x.x), x.y, w[t][i]);
        }
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) w[t][i] += __shfl_xor(w[t][i], d);
    // lane r16 = 4 t + i of a group writes key 16 t + 4 g + i
    if (r16 < 8) {
        float mine = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) mine = r16 == i ? w[i >> 2][i & 3] : mine;
        sums[wave][16 * (r16 >> 2) + 4 * g + (r16 & 3)] = mine;
    }
    __syncthreads();
    const int pos = (chunk - a.chunk_begin[s]) * a.chunk * kBlockTok + threadIdx.x;
    if ((int)threadIdx.x < a.chunk * kBlockTok && pos < L) {
        float sum = 0.f;
        for (int v = threadIdx.x >> 5; v < W; v += a.chunk) sum += sums[v][threadIdx.x & 31];
        const size_t o = ((size_t)s * kKvHeads + h) * (size_t)a.stride + pos;
        a.acc_out[o] = (a.acc_in ? a.acc_in[o] : 0.f) + sum;
    }
}

// ---------------------------------------------------------------------------
// Which tokens stay: one workgroup per (layer, sequence, kv head).  Accumulated
// weights are ordered as unsigned integers (evict_key); the key of the last one
// that stays comes from 3 passes over the row, 11, 11 and 10 of the key's bits
// each (histogram in LDS; integer atomics: any order, the same counts).  A
// token stays if its key is greater, or equal and among the first of the equal
// ones that still fit.  Sinks and recent tokens have no part in the choice.
// Wave w takes the w'th sixteenth of the row; REGS keys per thread stay in
// registers over the passes, 0: rows too long for that are read again.
// Bound by latency (one memory access, 14 barriers of 16 waves, the atomics of
// equal digits): 8 layers of 4096 tokens 11-12 us, 16 sequences of 5000 12 us
// (four passes of 8 bits over memory 13.2 and 14.2).
constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64, kSelRegs = 8, kSelBins = 2048;

// Greater weight -> greater key; NaN lowest; -0 as +0.
__device__ __forceinline__ uint32_t evict_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int REGS>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictSelectArgs a) {
    __shared__ uint32_t hist[kSelBins];
    __shared__ uint32_t sh_key, sh_need;
    __shared__ uint32_t wsum[2][kSelWaves];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int h = blockIdx.x % kKvHeads, j = blockIdx.x / kKvHeads % a.n_seqs, layer = blockIdx.x / kKvHeads / a.n_seqs;
    const size_t row = ((size_t)layer * a.call_seqs + a.seq0 + j) * kKvHeads + h;
    const float* acc = a.acc + row * (size_t)a.stride;
    float* acc_out = a.acc_out ? a.acc_out + row * (size_t)a.stride : nullptr;
    int32_t* kept = a.kept + row * (size_t)a.budget;
    const int L = a.len[j];
    const int n_keep = min(L, a.budget);
    const int lo = min(a.n_sink, L), hi = max(lo, L - a.n_recent);  // the choice: [lo, hi)
    const int n_pick = L <= a.budget ? hi - lo : a.budget - a.n_sink - a.n_recent;
    const int steps = (L + kSelThreads - 1) / kSelThreads;  // tokens per thread
    const int first = wave * steps * 64 + lane;             // the thread's: first + 64 k
    float x[REGS > 0 ? REGS : 1];
    if constexpr (REGS > 0) {
#pragma unroll
        for (int k = 0; k < REGS; k++) x[k] = k < steps && first + 64 * k < L ? acc[first + 64 * k] : 0.f;
    }
    // f(token, weight) for the thread's tokens in order, all lanes at once (the
    // token may be L or more)
    const auto walk = [&](auto f) {
        if constexpr (REGS > 0) {
#pragma unroll
            for (int k = 0; k < REGS; k++)
                if (k < steps) f(first + 64 * k, x[k]);
        } else {
            for (int k = 0; k < steps; k += 4) {
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = k + i < steps && first + 64 * (k + i) < L ? acc[first + 64 * (k + i)] : 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (k + i < steps) f(first + 64 * (k + i), y[i]);
            }
        }
    };
    uint32_t key = 0, need = 0;  // keys > key stay, and the first `need` equal ones
    if (n_pick < hi - lo) {
        if (n_pick == 0) {
            key = 0xFFFFFFFFu;
        } else {
            need = (uint32_t)n_pick;
#pragma unroll
            for (int pass = 0; pass < 3; pass++) {
                constexpr int kShift[3] = {21, 10, 0};
                const int shift = kShift[pass];
                const uint32_t digits = pass < 2 ? 2048 : 1024;
                for (int i = t; i < kSelBins; i += kSelThreads) hist[i] = 0;
                __syncthreads();
                walk([&](int i, float w) {
                    const uint32_t k = evict_key(w);
                    if (i >= lo && i < hi && (pass == 0 || (k ^ key) >> (pass == 1 ? 21 : 10) == 0))
                        __hip_atomic_fetch_add(&hist[(k >> shift) & (digits - 1)], 1u, __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_WORKGROUP);
                });
                __syncthreads();
                // thread t holds digits 2047 - 2 t and 2046 - 2 t, greatest first
                const uint32_t c0 = hist[kSelBins - 1 - 2 * t], c1 = hist[kSelBins - 2 - 2 * t];
                uint32_t before = c0 + c1;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const uint32_t o = __shfl_up(before, d);
                    if (lane >= d) before += o;
                }
                if (lane == 63) wsum[0][wave] = before;
                __syncthreads();
                before -= c0 + c1;
#pragma unroll
                for (int w = 0; w < kSelWaves; w++) before += w < wave ? wsum[0][w] : 0;
                if (before < need && need <= before + c0) {
                    sh_key = key | (uint32_t)(kSelBins - 1 - 2 * t) << shift;
                    sh_need = need - before;
                }
                before += c0;
                if (before < need && need <= before + c1) {
                    sh_key = key | (uint32_t)(kSelBins - 2 - 2 * t) << shift;
                    sh_need = need - before;
                }
                __syncthreads();
                key = sh_key;
                need = sh_need;
            }
        }
    }
    const bool all = n_pick >= hi - lo;
    const auto above = [&](int i, float w) { return i < L && (i < lo || i >= hi || all || evict_key(w) > key); };
    const auto equal = [&](int i, float w) { return i >= lo && i < hi && !all && evict_key(w) == key; };
    uint32_t n_above = 0, n_equal = 0;  // of the wave's tokens, then of all before the one at hand
    walk([&](int i, float w) {
        n_above += __popcll(__builtin_amdgcn_ballot_w64(above(i, w)));
        n_equal += __popcll(__builtin_amdgcn_ballot_w64(equal(i, w)));
    });
    __syncthreads();
    if (lane == 0) wsum[0][wave] = n_above, wsum[1][wave] = n_equal;
    __syncthreads();
    n_above = n_equal = 0;
#pragma unroll
    for (int w = 0; w < kSelWaves; w++) {
        n_above += w < wave ? wsum[0][w] : 0;
        n_equal += w < wave ? wsum[1][w] : 0;
    }
    const uint64_t below = (1ull << lane) - 1ull;
    walk([&](int i, float w) {
        const bool ab = above(i, w), eq = equal(i, w);
        const uint64_t ab_m = __builtin_amdgcn_ballot_w64(ab), eq_m = __builtin_amdgcn_ballot_w64(eq);
        const uint32_t rank = n_equal + __popcll(eq_m & below);
        const uint32_t at = n_above + __popcll(ab_m & below) + min(rank, need);
        if (ab || (eq && rank < need)) {
            kept[at] = i;
            if (acc_out) acc_out[at] = w;
        }
        n_above += __popcll(ab_m);
        n_equal += __popcll(eq_m);
    });
    for (uint32_t i = n_keep + t; i < (uint32_t)a.budget; i += kSelThreads) kept[i] = -1;  // (a budget near 2^31)
    if (acc_out)
        for (int i = n_keep + t; i < L; i += kSelThreads) acc_out[i] = 0.f;
}

// Moves the kept rows: one workgroup = one (layer, K|V, kv head) unit of a new
// block.  Rows of 8-bit blocks become bf16(i s).  Slots past the new length
// are left as they were.  Bound by memory, 512 B at a time from anywhere: 1501
// of 5000 tokens of 16 sequences 34 us, 5.8 TB/s read and written.
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictCopyArgs a) {
    const int per = a.p.n_layers * 2 * kKvHeads;
    const int i = blockIdx.x / per, u = blockIdx.x % per;
    const int h = u % kKvHeads, kv = (u / kKvHeads) & 1, lkv = u / kKvHeads, layer = lkv >> 1;
    const int s = find_seq(a.begin, a.n_seqs, i);
    const int b = i - a.begin[s];
    const int32_t* from = a.p.table + (size_t)a.src[s] * a.p.table_stride;
    const int id = a.p.table[(size_t)a.dst[s] * a.p.table_stride + b];
    const int32_t* kept = a.kept + (((size_t)layer * a.call_seqs + a.seq0 + s) * kKvHeads + h) * (size_t)a.budget;
    uint8_t* pool = a.p.pool + (int64_t)lkv * a.p.layer_kv_bytes;
    const uint8_t* q8 = a.p.q8 + (int64_t)lkv * a.p.q8_kv_bytes;
    const float* scales = a.p.scales + (int64_t)lkv * a.p.scale_kv;
    const int n = min(kBlockTok, a.new_len[s] - b * kBlockTok);
    const int part = threadIdx.x & 31;
    u32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int tok = j * 8 + (threadIdx.x >> 5);
        if (tok >= n) break;
        const int pos = kept[b * kBlockTok + tok];
        const size_t unit = (size_t)from[pos / kBlockTok] * kKvHeads + h;
        const int slot = pos % kBlockTok;
        if (pos / kBlockTok < a.n8[s]) {
            const uint8_t* src = q8 + unit * kQ8UnitBytes;
            const float scale = scales[unit];
            float f[8];
#pragma unroll
            for (int d = 0; d < 8; d++)
                f[d] = (float)(int8_t)src[kv ? q8_v_off(slot, part * 8 + d) : q8_k_off(slot, part * 8 + d)] * scale;
            x[j] = pack_bf16x8(f);
        } else {
            x[j] = *reinterpret_cast<const u32x4*>(pool + unit * kUnitBytes + slot * kHeadDim * 2 + part * 16);
        }
    }
    uint8_t* to = pool + ((size_t)id * kKvHeads + h) * kUnitBytes + part * 16;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int tok = j * 8 + (threadIdx.x >> 5);
        if (tok < n) *reinterpret_cast<u32x4*>(to + tok * kHeadDim * 2) = x[j];
    }
}

// ---------------------------------------------------------------------------

int launch_weights(const WeightsArgs& a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid(a.total_chunks * kKvHeads);
    if (weights_store(a.n_q)) {
        hipLaunchKernelGGL(weights_score_kernel<true>, grid, dim3(64 * weights_waves(true)), 0, st, a);
        hipLaunchKernelGGL(weights_sum_kernel, dim3(a.sum_chunks * kKvHeads), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL(weights_score_kernel<false>, grid, dim3(64 * weights_waves(false)), 0, st, a);
        hipLaunchKernelGGL(weights_again_kernel, grid, dim3(64 * weights_waves(false)), 0, st, a);
    }
    return (int)hipGetLastError();
}

int launch_evict_select(const EvictSelectArgs& a, void* stream) {
    const dim3 grid(a.n_layers * a.n_seqs * kKvHeads), block(kSelThreads);
    int32_t longest = 0;
    for (int32_t j = 0; j < a.n_seqs; j++) longest = std::max(longest, a.len[j]);
    if (longest <= kSelRegs * kSelThreads)
        hipLaunchKernelGGL(evict_select_kernel<kSelRegs>, grid, block, 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(evict_select_kernel<0>, grid, block, 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int launch_evict_copy(const EvictCopyArgs& a, void* stream) {
    const unsigned grid = (unsigned)a.n_blocks * a.p.n_layers * 2 * kKvHeads;
    hipLaunchKernelGGL(evict_copy_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

}  // namespace kvc
