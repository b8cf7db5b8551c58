// kvc_evict_kernels.h -- kernels of eviction by accumulated attention weight:
// the weights that query rows give every cached token, the choice of the
// tokens that stay, and the move of their rows.  Included by kvc_kernels.hip.
#pragma once

namespace kvc {

// ---------------------------------------------------------------------------
// Attention weights, first launch: scores of all rows of a kv head (row 4 i +
// g = query i, q head g of the group) against the keys of a chunk of
// kWeightsChunk blocks, one block per wave.  The block's K sits in registers
// as A operand (keys x dims; 8-bit blocks as exact bf16 integers, scaled
// after the product) and the rows pass by in tiles of 16 (B operand).  Scores
// go to the workspace in the log2 domain, -infinity where the row does not see
// the key, with the chunk's (max, sum 2^(s - max)) per row; the second launch
// needs every chunk's before it can normalise any weight.
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

__global__ __launch_bounds__(256) void weights_score_kernel(WeightsArgs a) {
    // (max, sum) of each wave's block and row
    __shared__ float2 ml[kWeightsChunk][kWeightsMaxQ * kGroup];
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunk = blockIdx.x >> 2, h = blockIdx.x & 3;
    const int s = find_seq(a.chunk_begin, a.n_seqs, chunk);
    const int L = a.kv_len[s], R = a.n_q * kGroup;
    const int nb = (L + kBlockTok - 1) / kBlockTok;
    const int b = (chunk - a.chunk_begin[s]) * kWeightsChunk + wave;
    const float none = -__builtin_inff();
    if (b < nb) {
        const int id = a.c.table[(size_t)a.slot[s] * a.c.table_stride + b];
        const bool q8 = b < a.n8[s];
        u32x4 kf[2][8];
        weights_load_k(kf, a.c, id, h, q8, lane);
        const float scale = q8 ? a.scale_log2 * a.c.ks[(size_t)id * kKvHeads + h] : a.scale_log2;
        float* out = a.scores + ((size_t)h * a.total_blocks + a.block_begin[s] + b) * R * kBlockTok;
        for (int r0 = 0; r0 < R; r0 += 16) {
            const int row = r0 + r16;
            const int rc = min(row, R - 1);
            const uint16_t* q = a.q + (((size_t)s * a.n_q + (rc >> 2)) * kQHeads + h * kGroup + (rc & 3)) * kHeadDim + 8 * g;
            u32x4 qf[8];
#pragma unroll
            for (int ks = 0; ks < 8; ks++) qf[ks] = *reinterpret_cast<const u32x4*>(q + 32 * ks);
            f32x4 st[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int ks = 0; ks < 8; ks++)
#pragma unroll
                for (int t = 0; t < 2; t++)
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kf[t][ks]), as_bf16x8(qf[ks]), st[t], 0, 0, 0);
            // lane: keys 16 t + 4 g + i of row `row`
            const int last = L - a.n_q + (rc >> 2);  // last key the row sees
            float mx = none;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    st[t][i] = b * kBlockTok + 16 * t + 4 * g + i <= last ? st[t][i] * scale : none;
                    mx = fmaxf(mx, st[t][i]);
                }
            mx = max_xor16(mx);
            mx = max_xor32(mx);
            float l = 0.f;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) l += fast_exp2(st[t][i] - fmaxf(mx, kNegBig));  // 0 for -infinity
            l = sum_xor16(l);
            l = sum_xor32(l);
            if (row < R) {
#pragma unroll
                for (int t = 0; t < 2; t++)
                    *reinterpret_cast<f32x4*>(out + (size_t)row * kBlockTok + 16 * t + 4 * g) = st[t];
                if (g == 0) ml[wave][row] = make_float2(fmaxf(mx, kNegBig), l);
            }
        }
    } else {
        for (int r = lane; r < R; r += 64) ml[wave][r] = make_float2(kNegBig, 0.f);
    }
    __syncthreads();
    float2* stats = reinterpret_cast<float2*>(a.stats) + ((size_t)h * a.total_chunks + chunk) * R;
    for (int r = threadIdx.x; r < R; r += 256) {
        float m = kNegBig, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWeightsChunk; w++) m = fmaxf(m, ml[w][r].x);
#pragma unroll
        for (int w = 0; w < kWeightsChunk; w++) l = fmaf(fast_exp2(ml[w][r].x - m), ml[w][r].y, l);
        stats[r] = make_float2(m, l);
    }
}

// Second launch: one workgroup = kWsumBlocks blocks of one kv head.  It folds
// the chunks' row statistics (each thread takes every 256 / R'th chunk of a
// row), then thread (key, block) sums its key's weights over the rows in
// order and adds them to the accumulator: no atomics, the same bits each time.
__global__ __launch_bounds__(256) void weights_sum_kernel(WeightsArgs a) {
    __shared__ float2 row_ml[kWeightsMaxQ * kGroup];
    __shared__ float2 part[256];
    const int t = threadIdx.x;
    const int item = blockIdx.x >> 2, h = blockIdx.x & 3;
    const int s = find_seq(a.sum_begin, a.n_seqs, item);
    const int L = a.kv_len[s], R = a.n_q * kGroup;
    const int nb = (L + kBlockTok - 1) / kBlockTok;
    const int nc = a.chunk_begin[s + 1] - a.chunk_begin[s];
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + ((size_t)h * a.total_chunks + a.chunk_begin[s]) * R;
    int lanes = 256;  // threads per row: a power of two
    while (lanes > 1 && lanes * R > 256) lanes >>= 1;
    const int rows = 256 / lanes;
    for (int r0 = 0; r0 < R; r0 += rows) {
        const int r = r0 + t / lanes;
        float m = kNegBig, l = 0.f;
        if (r < R)
            for (int k = t % lanes; k < nc; k += lanes) {
                const float2 x = stats[(size_t)k * R + r];
                const float mn = fmaxf(m, x.x);
                l = fmaf(l, fast_exp2(m - mn), x.y * fast_exp2(x.x - mn));
                m = mn;
            }
        part[t] = make_float2(m, l);
        __syncthreads();
        for (int d = lanes >> 1; d > 0; d >>= 1) {
            if (t % lanes < d) {
                const float2 x = part[t], y = part[t + d];
                const float mn = fmaxf(x.x, y.x);
                part[t] = make_float2(mn, fmaf(x.y, fast_exp2(x.x - mn), y.y * fast_exp2(y.x - mn)));
            }
            __syncthreads();
        }
        if (t % lanes == 0 && r < R) row_ml[r] = make_float2(part[t].x, 1.0f / part[t].y);
        __syncthreads();
    }
    const int b = (item - a.sum_begin[s]) * kWsumBlocks + (t >> 5), key = t & 31;
    const int pos = b * kBlockTok + key;
    if (b >= nb || pos >= L) return;
    const float* sc = a.scores + ((size_t)h * a.total_blocks + a.block_begin[s] + b) * R * kBlockTok + key;
    float w = 0.f;
#pragma unroll 8
    for (int r = 0; r < R; r++) {
        const float2 x = row_ml[r];
        w = fmaf(fast_exp2(sc[(size_t)r * kBlockTok] - x.x), x.y, w);
    }
    const size_t o = ((size_t)s * kKvHeads + h) * (size_t)a.stride + pos;
    a.acc_out[o] = (a.acc_in ? a.acc_in[o] : 0.f) + w;
}

// ---------------------------------------------------------------------------
// Which tokens stay: one workgroup per (layer, sequence, kv head).  Accumulated
// weights are ordered as unsigned integers (evict_key); the value of the last
// one that stays comes from 4 passes over the row, 8 bits of the key each
// (histogram in LDS), and the row is then walked once more in order: a token
// stays if its key is greater, or equal and among the first of the equal ones
// that still fit.  Sinks and recent tokens have no part in the choice.
constexpr int kSelThreads = 1024;

// Greater weight -> greater key; NaN lowest; -0 as +0.
__device__ __forceinline__ uint32_t evict_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictSelectArgs a) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t sh_key, sh_need;
    __shared__ int wsum[2][kSelThreads / 64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int h = blockIdx.x % kKvHeads, j = blockIdx.x / kKvHeads % a.n_seqs, layer = blockIdx.x / kKvHeads / a.n_seqs;
    const size_t row = ((size_t)layer * a.call_seqs + a.seq0 + j) * kKvHeads + h;
    const float* acc = a.acc + row * (size_t)a.stride;
    float* acc_out = a.acc_out ? a.acc_out + row * (size_t)a.stride : nullptr;
    int32_t* kept = a.kept + row * (size_t)a.budget;
    const int L = a.len[j];
    const int n_keep = min(L, a.budget);
    const int lo = min(a.n_sink, L), hi = max(lo, L - a.n_recent);  // the choice: [lo, hi)
    const int n_pick = L <= a.budget ? hi - lo : a.budget - a.n_sink - a.n_recent;
    uint32_t key = 0, need = 0;  // keys > key stay, and the first `need` equal ones
    if (n_pick < hi - lo) {
        if (n_pick == 0) {
            key = 0xFFFFFFFFu;
        } else {
            uint32_t left = (uint32_t)n_pick;
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int i = t; i < 256; i += kSelThreads) hist[i] = 0;
                __syncthreads();
                for (int i = lo + t; i < hi; i += kSelThreads) {
                    const uint32_t k = evict_key(acc[i]);
                    if (shift == 24 || (k >> (shift + 8)) == (key >> (shift + 8)))
                        __hip_atomic_fetch_add(&hist[(k >> shift) & 255], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                }
                __syncthreads();
                if (wave == 0) {
                    // lane holds digits 255 - 4 lane .. 252 - 4 lane, greatest first
                    uint32_t c[4], sum = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        c[i] = hist[255 - 4 * lane - i];
                        sum += c[i];
                    }
                    uint32_t before = sum;  // inclusive prefix over the lanes
                    for (int d = 1; d < 64; d <<= 1) {
                        const uint32_t o = __shfl_up(before, d);
                        if (lane >= d) before += o;
                    }
                    before -= sum;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (before < left && left <= before + c[i]) {
                            sh_key = key | (uint32_t)(255 - 4 * lane - i) << shift;
                            sh_need = left - before;
                        }
                        before += c[i];
                    }
                }
                __syncthreads();
                key = sh_key;
                left = sh_need;
                __syncthreads();
            }
            need = left;
        }
    }
    const bool all = n_pick >= hi - lo;
    int n_out = 0;
    uint32_t n_equal = 0;
    for (int i0 = 0; i0 < L; i0 += kSelThreads) {
        const int i = i0 + t;
        const float x = i < L ? acc[i] : 0.f;
        const bool forced = i < L && (i < lo || i >= hi || all);
        const uint32_t k = evict_key(x);
        const bool pick = i < L && !forced;
        const bool equal = pick && k == key && need > 0;
        const uint64_t eq = __builtin_amdgcn_ballot_w64(equal);
        const uint64_t below = (1ull << lane) - 1ull;
        if (lane == 0) wsum[0][wave] = __popcll(eq);
        __syncthreads();
        uint32_t rank = n_equal + __popcll(eq & below);
        for (int w = 0; w < kSelThreads / 64; w++) {
            if (w < wave) rank += wsum[0][w];
            n_equal += wsum[0][w];
        }
        const bool stay = forced || (pick && k > key) || (equal && rank < need);
        const uint64_t st = __builtin_amdgcn_ballot_w64(stay);
        if (lane == 0) wsum[1][wave] = __popcll(st);
        __syncthreads();
        int at = n_out + __popcll(st & below);
        for (int w = 0; w < kSelThreads / 64; w++) {
            if (w < wave) at += wsum[1][w];
            n_out += wsum[1][w];
        }
        if (stay) {
            kept[at] = i;
            if (acc_out) acc_out[at] = x;
        }
        __syncthreads();
    }
    for (int i = n_keep + t; i < a.budget; i += kSelThreads) kept[i] = -1;
    if (acc_out)
        for (int i = n_keep + t; i < L; i += kSelThreads) acc_out[i] = 0.f;
}

// Moves the kept rows: one workgroup = one (layer, K|V, kv head) unit of a new
// block.  Rows of 8-bit blocks become bf16(i s).  Slots past the new length
// are left as they were.
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
    hipLaunchKernelGGL(weights_score_kernel, dim3(a.total_chunks * kKvHeads), dim3(256), 0, st, a);
    hipLaunchKernelGGL(weights_sum_kernel, dim3(a.sum_chunks * kKvHeads), dim3(256), 0, st, a);
    return (int)hipGetLastError();
}

int launch_evict_select(const EvictSelectArgs& a, void* stream) {
    hipLaunchKernelGGL(evict_select_kernel, dim3(a.n_layers * a.n_seqs * kKvHeads), dim3(kSelThreads), 0,
                       (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int launch_evict_copy(const EvictCopyArgs& a, void* stream) {
    const unsigned grid = (unsigned)a.n_blocks * a.p.n_layers * 2 * kKvHeads;
    hipLaunchKernelGGL(evict_copy_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

}  // namespace kvc
