// kvc_prefill_q8_kernels.h -- causal chunked prefill over sequences that start
// with 8-bit blocks.  Included by kvc_kernels.hip, whose helpers it uses.
#pragma once

namespace kvc {

// ---------------------------------------------------------------------------
// One workgroup holds 64 query rows of one kv head: 4 waves, wave g those of q
// head g, in two halves of 32 rows.  Keys pass by one 32-token block a step:
//   S^T[32 keys x 32 rows] = K . Q^T          (A = K rows from LDS, B = Q)
//   P^T = 2^(c ks S^T - m) vs                 (bf16; fp32 sums of 2^(..) beside)
//   O^T[256 dims x 32 rows] += V^T . P^T      (A = V^T from LDS)
// with v_mfma_f32_32x32x16_bf16.  A wave alone on its SIMD has 512 registers: O
// (256), Q (128), S and P of 64 rows.  An operand fragment read from LDS
// serves 64 (K) or 32 (V^T) rows, so the LDS pipe is busy 1536 cycles a step
// beside 2048 of the matrix pipe, and the first half's P.V products cover the
// second half's softmax.  A lane works on one row (l % 32) of a half and 16 of
// the block's keys, in an order in which P^T leaves the S^T accumulator as B
// operand: lane half f, product j takes keys 16 j + 4 f + {0..3, 8..11}, the
// order in which V pieces hold their tokens.
//
// 8-bit blocks: pieces go from memory straight to LDS as they are
// (global_load_lds, 3 steps ahead of their use, no registers); during step b
// each wave turns its own pieces of block b + 1 into bf16 integers (exact) in
// the tile that step b + 1 reads.  bf16 blocks (a sequence's tail and the
// chunk) are copied into that tile directly, one step ahead.  One barrier a
// step.
//
// Work split: all (sequence, kv head, 64 rows) items' blocks in one line, cut
// into equal runs, one per workgroup, so that ragged batches keep every CU busy
// to the end.  A run that holds a whole item writes its output; the others
// leave unnormalised partials (at most 2 per workgroup) for
// prefill_q8_combine_kernel.
constexpr int kP8Raw = 4;  // 8-bit blocks in flight
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef const __attribute__((address_space(4))) int32_t* const_i32;
typedef const __attribute__((address_space(4))) float* const_f32;

struct PrefillQ8Smem {
    uint16_t k[2][kBlockTok * kHeadDim];  // rows, 16-B chunks swizzled by p8_kswz
    uint16_t v[2][kBlockTok * kHeadDim];  // 8-bit block: V^T fragments in order; bf16: rows swizzled by p8_vswz
    uint8_t raw[kP8Raw][2 * kQ8UnitBytes];
};

// K fragment reads take one chunk of 32 rows, V^T reads 64 B of 8 rows.
__device__ __forceinline__ int p8_kswz(int r) { return r & 7; }
__device__ __forceinline__ int p8_vswz(int r) { return (r & 7) << 2; }

// Blocks of row block rb of a sequence whose first row sits at pos0.
__device__ __forceinline__ int p8_blocks(int pos0, int n_q, int rb) {
    return (pos0 + min((rb + 1) * kP8Rows, n_q) + kBlockTok - 1) / kBlockTok;
}

// The item that unit `at` of the line falls into.
struct P8Item {
    int s, h, rb;
    int begin, n;  // its first unit, its blocks
};
__device__ __forceinline__ P8Item p8_find(const PrefillQ8Args& a, int at) {
    P8Item it;
    it.s = find_seq(a.begin, a.n_seqs, at);
    const int per_head = (a.begin[it.s + 1] - a.begin[it.s]) / kKvHeads;
    const int off = at - a.begin[it.s];
    it.h = off / per_head;
    it.begin = a.begin[it.s] + it.h * per_head;
    it.rb = 0;
    it.n = p8_blocks(a.q_pos0[it.s], a.n_q, 0);
    while (at >= it.begin + it.n) {
        it.begin += it.n;
        it.n = p8_blocks(a.q_pos0[it.s], a.n_q, ++it.rb);
    }
    return it;
}

template <bool FINE>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void prefill_q8_kernel(PrefillQ8Args a) {
    __shared__ __align__(1024) PrefillQ8Smem sm;
    const int wg = (blockIdx.x & 7) * a.per_xcd + (blockIdx.x >> 3);
    const int u_begin = wg * a.per_wg, u_end = min(u_begin + a.per_wg, a.total);
    if (wg >= a.n_wgs || u_begin >= u_end) return;
    const int lane = threadIdx.x & 63, r32 = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = wave & 3, rg = wave >> 2;  // q head of the group, half of the rows
    const float c = fabsf(a.scale_log2);
    const uint32_t qflip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    const uint32_t k0 = lds_addr(&sm.k[0][0]), v0 = lds_addr(&sm.v[0][0]), raw0 = lds_addr(&sm.raw[0][0]);
    constexpr uint32_t kTile = kBlockTok * kHeadDim * 2;

    for (int at = u_begin; at < u_end;) {
        const P8Item it = p8_find(a, at);
        const int s = it.s, h = it.h;
        const int b0 = at - it.begin, b1 = min(it.n, u_end - it.begin);
        const int pos0 = a.q_pos0[s], row0 = it.rb * kP8Rows;
        const int rows = min(kP8Rows, a.n_q - row0);
        const int kmax = pos0 + row0 + rows;  // keys [0, kmax) are seen
        const int n8 = a.n8[s];
        // block ids and scales come through scalar loads (a vector load in the
        // loop would have its wait drain the copies in flight): id[i] is block b
        // + i's, ks / vs block b's and the next one's
        const const_i32 trow = (const_i32)(a.c.table + (size_t)a.slot[s] * a.c.table_stride);
        int id[kP8Raw];
#pragma unroll
        for (int i = 0; i < kP8Raw; i++) id[i] = trow[min(b0 + i, b1 - 1)];
        const auto scale_of = [&](const float* scales, int b, int id) {
            return b < n8 ? ((const_f32)scales)[id * kKvHeads + h] : 1.f;
        };

        // pieces of an 8-bit block into the ring: wave w its 64 of K and of V
        const auto issue_raw = [&](int b, int id) {
            const size_t unit = (size_t)id * kKvHeads + h;
            const uint32_t to = raw0 + (b & (kP8Raw - 1)) * (2 * kQ8UnitBytes) + wave * 1024;
            lds_dma16s(a.c.k8 + unit * kQ8UnitBytes + wave * 1024, lane * 16, to);
            lds_dma16s(a.c.v8 + unit * kQ8UnitBytes + wave * 1024, lane * 16, to + kQ8UnitBytes);
        };
        // rows of a bf16 block into tile b & 1: wave w rows 4 w .. + 3; rows past
        // the last key repeat it (finite where it is, and their weight is 0)
        const auto issue_rows = [&](int b, int id) {
            const size_t unit = ((size_t)id * kKvHeads + h) * kBlockTok * kHeadDim;
            const int last = kmax - 1 - b * kBlockTok;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int r0 = 4 * wave + 2 * i, r = r0 + hf;
                const uint32_t from = min(r, last) * 512;
                const uint32_t to = (b & 1) * kTile + r0 * 512;
                lds_dma16s(a.c.kpool + unit, from + 16 * (r32 ^ p8_kswz(r)), k0 + to);
                lds_dma16s(a.c.vpool + unit, from + 16 * (r32 ^ p8_vswz(r)), v0 + to);
            }
        };
        // the wave's pieces of 8-bit block b -> tile b & 1
        const auto convert = [&](int b, int lane) {
            const int cc = lane & 15, gg = lane >> 4;
            const int e = wave;
            {
                const uint32_t from = raw0 + (b & (kP8Raw - 1)) * (2 * kQ8UnitBytes) + e * 1024 + lane * 16;
                const u32x4 kp = lds_load16(from, 0), vp = lds_load16(from, kQ8UnitBytes);
                const int kr = 16 * (e >> 2) + cc, ch = 8 * (e & 3) + 2 * gg;
                u32x4 x0, x1;
                const auto widen = [&](const u32x4& p) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const u32x2 lo = i8x4_to_bf16(p[i]), hi = i8x4_to_bf16(p[2 + i]);
                        x0[2 * i] = lo[0];
                        x0[2 * i + 1] = lo[1];
                        x1[2 * i] = hi[0];
                        x1[2 * i + 1] = hi[1];
                    }
                };
                widen(kp);
                u32x4* kd = reinterpret_cast<u32x4*>(&sm.k[b & 1][kr * kHeadDim]);
                kd[ch ^ p8_kswz(kr)] = x0;
                kd[(ch + 1) ^ p8_kswz(kr)] = x1;
                widen(vp);
                // fragment (dt = e, j = gg / 2), lanes 32 (gg % 2) + cc and + 16
                u32x4* vd = reinterpret_cast<u32x4*>(&sm.v[b & 1][0]) + (e * 2 + (gg >> 1)) * 64 + 32 * (gg & 1) + cc;
                vd[0] = x0;
                vd[16] = x1;
            }
        };

        // everything the last item left in LDS has been read
        __syncthreads();
        const int n_raw = min(b1, n8);  // blocks [b0, n_raw) of the run are 8-bit ones
#pragma unroll
        for (int i = 0; i < kP8Raw - 1; i++)
            if (b0 + i < n_raw) issue_raw(b0 + i, id[i]);
        if (b0 >= n8) issue_rows(b0, id[0]);

        {
            constexpr int H = 1;
            f32x16 o[H][8];
            float m_run[H], l_run[H];
            bf16x8_t qb[H][16];
#pragma unroll
            for (int x = 0; x < H; x++) {
                const int r = row0 + min(32 * rg + r32, rows - 1);
                const uint16_t* q = a.q + (((size_t)s * a.n_q + r) * kQHeads + h * kGroup + g) * kHeadDim + 8 * hf;
#pragma unroll
                for (int ks = 0; ks < 16; ks++) {
                    u32x4 w = *reinterpret_cast<const u32x4*>(q + 16 * ks);
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] ^= qflip;
                    qb[x][ks] = as_bf16x8(w);
                }
#pragma unroll
                for (int dt = 0; dt < 8; dt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[x][dt][i] = 0.f;
                m_run[x] = kNegBig;
                l_run[x] = 0.f;
            }
            if (b0 < n_raw) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                convert(b0, lane);
            }
            float ks_next = scale_of(a.c.ks, b0, id[0]), vs_next = scale_of(a.c.vs, b0, id[0]);
            // block b of the run, an 8-bit one or a bf16 one
            const auto step = [&](auto q8_, int b) {
                constexpr bool q8 = decltype(q8_)::value != 0;
                const float kscale = ks_next, vscale = vs_next;
                // tile b is written, the last reader of tile b + 1 is done
                if constexpr (q8)
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                else
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (b + kP8Raw - 1 < n_raw) issue_raw(b + kP8Raw - 1, id[kP8Raw - 1]);
                if (!(q8 && b + 1 < n8) && b + 1 < b1) issue_rows(b + 1, id[1]);
                ks_next = q8 ? scale_of(a.c.ks, b + 1, id[1]) : 1.f;
                vs_next = q8 ? scale_of(a.c.vs, b + 1, id[1]) : 1.f;
#pragma unroll
                for (int i = 0; i + 1 < kP8Raw; i++) id[i] = id[i + 1];
                id[kP8Raw - 1] = trow[min(b + kP8Raw, b1 - 1)];
                const uint32_t toff = (b & 1) * kTile;
                // lane-dependent addresses are made anew each step: kept over the
                // loop they would cost registers that Q and S need
                int ln = lane;
                asm volatile("" : "+v"(ln));
                const int r32 = ln & 31, hf = ln >> 5;
                // K fragment ks: row r32, chunk 2 ks + hf: kaddr[ks & 3] + 128 (ks >> 2)
                uint32_t kaddr[4];
#pragma unroll
                for (int j = 0; j < 4; j++) kaddr[j] = k0 + toff + r32 * 512 + 16 * ((2 * j + hf) ^ p8_kswz(r32));
                f32x16 st[H];
                {
                    bf16x8_t kf[4];
                    const auto read = [&](int ks) { return as_bf16x8(lds_load16(kaddr[ks & 3], 128 * (ks >> 2))); };
#pragma unroll
                    for (int ks = 0; ks < 4; ks++) kf[ks] = read(ks);
                    constexpr f32x16 zero = {};
#pragma unroll
                    for (int ks = 0; ks < 16; ks++) {
                        const bf16x8_t ka = kf[ks & 3];
                        if (ks + 4 < 16) kf[ks & 3] = read(ks + 4);
#pragma unroll
                        for (int x = 0; x < H; x++)
                            st[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka, qb[x][ks], ks ? st[x] : zero, 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(kSgDsRead, 4, 0);
#pragma unroll
                    for (int ks = 0; ks < 16; ks++) {
                        if (ks + 4 < 16) __builtin_amdgcn_sched_group_barrier(kSgDsRead, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(kSgMfma, 1, 0);
                    }
                }
                const float cq = c * kscale;  // >= 0 (or NaN)
                bf16x8_t pb[H][2], pl[H][2], pt[H][2];
                // lane: keys 8 (i / 4) + 4 hf + i % 4 of row r32 of half x.  A block
                // that the half's rows see whole keeps raw scores: the maximum is
                // scaled once and the scale enters the exponent through an FMA
                const auto softmax = [&](int x) {
                    const bool full = b * kBlockTok + kBlockTok - 1 <= pos0 + row0 + 32 * rg && (b + 1) * kBlockTok <= kmax;
                    if (!full) {
                        asm volatile("");
                        const int qpos = min(pos0 + row0 + 32 * rg + r32, kmax - 1);
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            st[x][i] = b * kBlockTok + 8 * (i >> 2) + 4 * hf + (i & 3) <= qpos ? st[x][i] * cq : kNegBig;
                    }
                    const float cs = full ? cq : 1.f;
                    float mx = st[x][0];
#pragma unroll
                    for (int i = 1; i < 16; i++) mx = fmaxf(mx, st[x][i]);
                    mx = max_xor32(mx);
                    mx = full ? mx * cq : mx;
                    if (__builtin_amdgcn_ballot_w64(mx > m_run[x] + kRescaleSlack) != 0) {
                        const bool up = mx > m_run[x] + kRescaleSlack;
                        const float cr = up ? fast_exp2(m_run[x] - mx) : 1.f;
                        m_run[x] = up ? mx : m_run[x];
                        l_run[x] *= cr;
#pragma unroll
                        for (int dt = 0; dt < 8; dt++) o[x][dt] *= cr;
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        u32x4 w, wl = {}, wt = {};
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            float y = fast_exp2(fmaf(st[x][8 * j + 2 * i], cs, -m_run[x]));
                            float z = fast_exp2(fmaf(st[x][8 * j + 2 * i + 1], cs, -m_run[x]));
                            l_run[x] += y + z;
                            y *= vscale;
                            z *= vscale;
                            w[i] = cvt_pk_bf16(y, z);
                            if constexpr (FINE) {  // each difference is exact
                                y -= bf16lo(w[i]);
                                z -= bf16hi(w[i]);
                                wl[i] = cvt_pk_bf16(y, z);
                                wt[i] = cvt_pk_bf16(y - bf16lo(wl[i]), z - bf16hi(wl[i]));
                            }
                        }
                        pb[x][j] = as_bf16x8(w);
                        pl[x][j] = as_bf16x8(wl);
                        pt[x][j] = as_bf16x8(wt);
                    }
                };
                const auto products = [&](int x, auto&& read) {
                    bf16x8_t vf[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) vf[i] = read(i);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int dt = i >> 1, j = i & 1;
                        const bf16x8_t va = vf[i & 3];
                        if (i + 4 < 16) vf[i & 3] = read(i + 4);
                        o[x][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pb[x][j], o[x][dt], 0, 0, 0);
                        if constexpr (FINE) {
                            o[x][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pl[x][j], o[x][dt], 0, 0, 0);
                            o[x][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pt[x][j], o[x][dt], 0, 0, 0);
                        }
                    }
                    constexpr int kReads = q8 ? 1 : 2, kProducts = FINE ? 3 : 1;
                    __builtin_amdgcn_sched_group_barrier(kSgDsRead, 4 * kReads, 1);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        if (i + 4 < 16) __builtin_amdgcn_sched_group_barrier(kSgDsRead, kReads, 1);
                        __builtin_amdgcn_sched_group_barrier(kSgMfma, kProducts, 1);
                    }
                };
                const auto pv = [&](int x) {
                    if constexpr (q8) {
                        const uint32_t base = v0 + toff + ln * 16;
                        products(x, [&](int i) { return as_bf16x8(lds_load16(base, 1024 * i)); });
                    } else {
                        // V^T through the transposing read: 16-lane group G takes dims
                        // 32 dt + 16 (G & 1) .. + 15 of rows 16 j + 4 hf + 0..3 (+ 8); its
                        // lane J addresses row J / 4, dims 4 (J % 4)
                        const int J = ln & 15, vr = 4 * hf + (J >> 2);
                        const uint32_t vtr = v0 + toff + vr * 512 + 32 * ((ln >> 4) & 1) + 8 * (J & 3);
                        products(x, [&](int i) {
                            // 64-B piece dt of rows vr (+ 8, + 16 j), all of one r & 7
                            const uint32_t y = vtr + (((i >> 1) ^ (vr & 7)) << 6);
                            const u32x2 lo = lds_load_tr16(y, 8192 * (i & 1)), hi = lds_load_tr16(y, 8192 * (i & 1) + 4096);
                            return as_bf16x8(u32x4{lo[0], lo[1], hi[0], hi[1]});
                        });
                    }
                };
                softmax(0);
                if constexpr (H == 2) softmax(1);
                pv(0);
                if constexpr (H == 2) pv(1);
                // the next block's pieces; only copies issued after them are left
                if (q8 && b + 1 < n_raw) {
                    if (b + 3 < n_raw)
                        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
                    else if (b + 2 < n_raw)
                        asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
                    else
                        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    convert(b + 1, ln);
                }
            };
            int b = b0;
            for (; b < n_raw; b++) step(PfBuf<1>{}, b);
            for (; b < b1; b++) step(PfBuf<0>{}, b);
            const int part_slot = 2 * wg + (at > u_begin);
#pragma unroll
            for (int x = 0; x < H; x++) {
                l_run[x] = sum_xor32(l_run[x]);
                const int rl = 32 * rg + r32;
                if (b0 > 0 || b1 < it.n) {  // a part of the item's keys
                    float* part = a.part + (size_t)part_slot * kP8PartFloats;
                    float* acc = part + ((size_t)(2 * g + rg) * 32 * 64 + lane) * 4;
#pragma unroll
                    for (int dt = 0; dt < 8; dt++)
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            *reinterpret_cast<f32x4*>(acc + (dt * 4 + q) * 256) =
                                f32x4{o[x][dt][4 * q], o[x][dt][4 * q + 1], o[x][dt][4 * q + 2], o[x][dt][4 * q + 3]};
                    if (hf == 0)
                        *reinterpret_cast<float2*>(part + kP8PartAcc + ((2 * g + rg) * 32 + r32) * 2) =
                            make_float2(m_run[x], l_run[x]);
                } else if (rl < rows) {
                    const size_t orow = (((size_t)s * a.n_q + row0 + rl) * kQHeads + h * kGroup + g) * kHeadDim;
#pragma unroll
                    for (int dt = 0; dt < 8; dt++) {
                        uint2 gw[4];
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            gw[q] = a.gate ? *reinterpret_cast<const uint2*>(a.gate + orow + 32 * dt + 8 * q + 4 * hf)
                                           : make_uint2(0u, 0u);
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            float gs[4] = {1.f, 1.f, 1.f, 1.f};
                            if (a.gate) gate_factors(gw[q], a.gate_ref, gs);
                            const float A[4] = {o[x][dt][4 * q], o[x][dt][4 * q + 1], o[x][dt][4 * q + 2], o[x][dt][4 * q + 3]};
                            write_out(a.out, a.out_bf16, orow, 32 * dt + 8 * q + 4 * hf, a.gate != nullptr, gs, l_run[x], A);
                        }
                    }
                }
            }
        }
        at = it.begin + b1;
    }
}

// Folds the partials of an item that the line's cuts went through: out =
// sum(w_p acc_p) / sum(w_p l_p), w_p = 2^(m_p - max m).  64 workgroups per cut
// (those of a cut that is not its item's first have nothing to do); a wave
// takes 32 rows of a q head x 8 dims, as the parts stored them.
constexpr int kP8Fold = 8;  // parts requested at once
__global__ __launch_bounds__(256) void prefill_q8_combine_kernel(PrefillQ8Args a) {
    const int cut = (blockIdx.x >> 6) + 1;  // between workgroups cut - 1 and cut
    const int u = cut * a.per_wg;
    const P8Item it = p8_find(a, u);
    // the cut is the item's first inner one (u = it.begin: no part before it)
    if (it.begin >= u || it.begin < u - a.per_wg) return;
    const int unit = (blockIdx.x & 63) * 4 + (threadIdx.x >> 6);
    const int row_group = unit >> 5, dq = unit & 31;  // (q head, half), (dim tile, quarter)
    const int lane = threadIdx.x & 63, r32 = lane & 31, hf = lane >> 5;
    const int row0 = it.rb * kP8Rows, rows = min(kP8Rows, a.n_q - row0), rl = 32 * (row_group & 1) + r32;
    if (32 * (row_group & 1) >= rows) return;
    const int w0 = cut - 1, w1 = (it.begin + it.n - 1) / a.per_wg;  // workgroups with a part of it
    // the first has it as its last run, unless its runs begin with it
    const auto slot = [&](int w) { return 2 * w + (w == w0 && it.begin > w0 * a.per_wg ? 1 : 0); };
    const size_t orow =
        (((size_t)it.s * a.n_q + row0 + min(rl, rows - 1)) * kQHeads + it.h * kGroup + (row_group >> 1)) * kHeadDim;
    const int d0 = 32 * (dq >> 2) + 8 * (dq & 3) + 4 * hf;
    const uint2 gw = a.gate ? *reinterpret_cast<const uint2*>(a.gate + orow + d0) : make_uint2(0u, 0u);
    float m = kNegBig, l = 0.f;
    f32x4 A = {0.f, 0.f, 0.f, 0.f};
    for (int w = w0; w <= w1; w += kP8Fold) {
        float2 st[kP8Fold];
        f32x4 x[kP8Fold];
#pragma unroll
        for (int k = 0; k < kP8Fold; k++) {  // past the end: the last part again, not used
            const float* part = a.part + (size_t)slot(min(w + k, w1)) * kP8PartFloats;
            st[k] = *reinterpret_cast<const float2*>(part + kP8PartAcc + (row_group * 32 + r32) * 2);
            x[k] = *reinterpret_cast<const f32x4*>(part + ((size_t)(row_group * 32 + dq) * 64 + lane) * 4);
        }
        float mx = m;
#pragma unroll
        for (int k = 0; k < kP8Fold; k++) mx = fmaxf(mx, st[k].x);
        const float cr = fast_exp2(m - mx);
        m = mx;
        l *= cr;
        A *= cr;
#pragma unroll
        for (int k = 0; k < kP8Fold; k++) {
            if (w + k <= w1) {
                const float wt = fast_exp2(st[k].x - m);
                l = fmaf(wt, st[k].y, l);
                A += x[k] * wt;
            }
        }
    }
    if (rl >= rows) return;
    float gs[4] = {1.f, 1.f, 1.f, 1.f};
    if (a.gate) gate_factors(gw, a.gate_ref, gs);
    const float o[4] = {A[0], A[1], A[2], A[3]};
    write_out(a.out, a.out_bf16, orow, d0, a.gate != nullptr, gs, l, o);
}

int launch_prefill_q8(const PrefillQ8Args& a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const int grid = a.per_xcd * 8;
    if (a.out_bf16)
        hipLaunchKernelGGL(prefill_q8_kernel<false>, dim3(grid), dim3(512), 0, st, a);
    else
        hipLaunchKernelGGL(prefill_q8_kernel<true>, dim3(grid), dim3(512), 0, st, a);
    if (a.n_wgs > 1) hipLaunchKernelGGL(prefill_q8_combine_kernel, dim3((a.n_wgs - 1) * 64), dim3(256), 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace kvc
