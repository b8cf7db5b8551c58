// kvc_prefill_q8_kernels.h -- causal chunked prefill over sequences that start
// with 8-bit blocks.  Included by kvc_kernels.hip, whose helpers it uses.
#pragma once

namespace kvc {

// ---------------------------------------------------------------------------
// One workgroup holds 64 query rows of one kv head: 8 waves, wave g + 4 rg the
// 32 rows of half rg of q head g.  Keys pass by one 32-token block a step:
//   S^T[32 keys x 32 rows] = K . Q^T          (A = K rows from LDS, B = Q)
//   P^T = 2^(c ks S^T - m) vs                 (bf16; fp32 sums of 2^(..) beside)
//   O^T[256 dims x 32 rows] += V^T . P^T      (A = V^T from LDS)
// with v_mfma_f32_32x32x16_bf16; c is the softmax scale times log2(e), ks and vs
// the block's 8-bit scales (1 for a bf16 block).  The row maximum m moves only
// when a block exceeds it by more than kRescaleSlack.  bf16 output rounds P
// once (2^-8 of each weight, as the output is); fp32 output (FINE) takes P as
// three bf16 parts, 2^-26, in three products.  O (128) and Q (64 registers) stay
// in registers: at 2 waves per SIMD a lane has 256.  A lane works on one row and
// 16 of the block's keys, in an order in which P^T leaves the S^T accumulator as
// B operand: lane half f, product j takes keys 16 j + 4 f + {0..3, 8..11}, the
// order in which V pieces hold their tokens.
//
// Bounds: a step is 2048 cycles of products per SIMD (2 waves x 32 x 32), 304 KB
// of LDS access per CU, 1330 cycles by SQ_LDS_IDX_ACTIVE, and 1500 of VALU issue
// for softmax and widening.  Measured, 16 sequences of 128 rows over 256..6000
// keys: 150 us, 650 TFLOP/s, against 1260 of a large matrix product (the clock is
// near 1.7 GHz); the matrix pipe is busy 37 % of the cycles, VALU 27 %, LDS 24 %,
// and the two waves per SIMD spend 35 % of their time at waits and barriers.  The
// fold takes another 21 us.  FINE: 231 and 24 us.
//
// 8-bit blocks: pieces go from memory straight to LDS as they are
// (global_load_lds, 3 steps ahead of their use, no registers); during step b
// each wave turns its own pieces of block b + 1 into bf16 integers (exact) in
// the tile that step b + 1 reads.  bf16 blocks (a sequence's tail and the
// chunk) are copied into a tile directly, 3 steps ahead too.  One barrier a
// step.
//
// Work split: all (sequence, kv head, 64 rows) items' blocks in one line, cut
// into runs of like cost, one per workgroup (prefill_q8_split), so that ragged
// batches keep every CU busy to the end.  A run that holds a whole item writes
// its output; the others leave unnormalised partials (at most 2 per workgroup)
// for prefill_q8_combine_kernel.
constexpr int kP8Raw = 4;  // 8-bit blocks in flight
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef const __attribute__((address_space(4))) int32_t* const_i32;
typedef const __attribute__((address_space(4))) float* const_f32;

struct PrefillQ8Tile {
    uint16_t k[kBlockTok * kHeadDim];  // rows, 16-B chunks swizzled by p8_kswz
    uint16_t v[kBlockTok * kHeadDim];  // 8-bit block: V^T fragments in order; bf16: rows swizzled by p8_vswz
};
// 8-bit block b of a run is read from tile b & 1, its pieces pass through slot
// b & 3 of the ring.  The bf16 blocks n_raw + j of a run follow in 4 tiles: the
// ring's two, which are free first (the one without the last 8-bit block's
// slot, then the other), then the two tiles, first the one that block n_raw - 1
// does not sit in.
union PrefillQ8Smem {
    PrefillQ8Tile tile[4];
    struct {
        PrefillQ8Tile tile8[2];
        uint8_t raw[kP8Raw][2 * kQ8UnitBytes];
    };
};

// K fragment reads take one chunk of 32 rows, 16 rows (256 B, all banks) at a
// time; V^T reads 64 B of 4 rows.
__device__ __forceinline__ int p8_kswz(int r) { return r & 15; }
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
// (s0: a sequence at or before it)
__device__ __forceinline__ P8Item p8_find(const PrefillQ8Args& a, int s0, int at) {
    P8Item it;
    it.s = s0;
    while (a.begin[it.s + 1] <= at) it.s++;
    const int per_head = (a.begin[it.s + 1] - a.begin[it.s]) / kKvHeads;
    it.h = (at - a.begin[it.s]) / per_head;
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
    if (wg >= a.n_wgs) return;
    const int u_begin = a.cut[wg], u_end = a.cut[wg + 1];
    const int lane = threadIdx.x & 63, r32 = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = wave & 3, rg = wave >> 2;  // q head of the group, half of the rows
    const float c = fabsf(a.scale_log2);
    const uint32_t qflip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    const uint32_t lds0 = lds_addr(&sm), raw0 = lds_addr(&sm.raw[0][0]);
    constexpr uint32_t kTile = sizeof(PrefillQ8Tile), kTileV = kTile / 2;

    int s_at = a.seq_at[wg];
    for (int at = u_begin; at < u_end;) {
        const P8Item it = p8_find(a, s_at, at);
        s_at = it.s;
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
        // rows of a bf16 block into its tile: wave w rows 4 w .. + 3; rows past
        // the last key repeat it (finite where it is, and their weight is 0)
        const int n_raw = min(b1, n8);  // blocks [b0, n_raw) of the run are 8-bit ones
        const int n_raw0 = max(n_raw, b0);
        const auto tile_of = [&](int b) -> uint32_t {  // LDS address
            const int j = b - n_raw0;
            const int t = j < 0 ? b & 1 : (j & 3) < 2 ? 2 + (((((n_raw0 - 1) >> 1) & 1) ^ 1) ^ (j & 1)) : (n_raw0 & 1) ^ (j & 1);
            return lds0 + t * kTile;
        };
        // (4 copies)
        const auto issue_rows = [&](int b, int id) {
            const size_t unit = ((size_t)id * kKvHeads + h) * kBlockTok * kHeadDim;
            const int last = kmax - 1 - b * kBlockTok;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int r0 = 4 * wave + 2 * i, r = r0 + hf;
                const uint32_t from = min(r, last) * 512;
                const uint32_t to = tile_of(b) + r0 * 512;
                lds_dma16s(a.c.kpool + unit, from + 16 * (r32 ^ p8_kswz(r)), to);
                lds_dma16s(a.c.vpool + unit, from + 16 * (r32 ^ p8_vswz(r)), to + kTileV);
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
                u32x4* kd = reinterpret_cast<u32x4*>(&sm.tile[b & 1].k[kr * kHeadDim]);
                kd[ch ^ p8_kswz(kr)] = x0;
                kd[(ch + 1) ^ p8_kswz(kr)] = x1;
                widen(vp);
                // fragment (dt = e, j = gg / 2), lanes 32 (gg % 2) + cc and + 16
                u32x4* vd = reinterpret_cast<u32x4*>(&sm.tile[b & 1].v[0]) + (e * 2 + (gg >> 1)) * 64 + 32 * (gg & 1) + cc;
                vd[0] = x0;
                vd[16] = x1;
            }
        };

        // everything the last item left in LDS has been read
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kP8Raw - 1; i++)
            if (b0 + i < n_raw) issue_raw(b0 + i, id[i]);
        if (n_raw == b0 + 1 && n_raw < b1) issue_rows(n_raw, id[1]);
        if (n_raw <= b0) {
#pragma unroll
            for (int i = 0; i < 3; i++)
                if (b0 + i < b1) issue_rows(b0 + i, id[i]);
        }

        {
            f32x16 o[8];
            float m_run = kNegBig, l_run = 0.f;
            bf16x8_t qb[16];
            {
                const int r = row0 + min(32 * rg + r32, rows - 1);
                const uint16_t* q = a.q + (((size_t)s * a.n_q + r) * kQHeads + h * kGroup + g) * kHeadDim + 8 * hf;
#pragma unroll
                for (int ks = 0; ks < 16; ks++) {
                    u32x4 w = *reinterpret_cast<const u32x4*>(q + 16 * ks);
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] ^= qflip;
                    qb[ks] = as_bf16x8(w);
                }
#pragma unroll
                for (int dt = 0; dt < 8; dt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[dt][i] = 0.f;
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
                // tile b is written (bf16: only copies issued after its own are
                // left), the readers of the tiles that are written next are done
                if constexpr (q8) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                } else {
                    if (b + 2 < b1)
                        asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
                    else if (b + 1 < b1)
                        asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)" ::: "memory");
                    else
                        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                }
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (q8 && b + kP8Raw - 1 < n_raw) issue_raw(b + kP8Raw - 1, id[kP8Raw - 1]);
                if constexpr (q8) {
                    if (b + 2 == n_raw && n_raw < b1) issue_rows(n_raw, id[2]);
                    if (b + 1 == n_raw) {
                        if (b + 2 < b1) issue_rows(b + 2, id[2]);
                        if (b + 3 < b1) issue_rows(b + 3, id[3]);
                    }
                } else {
                    if (b + 3 < b1) issue_rows(b + 3, id[3]);
                }
                // lane-dependent addresses are made anew each step: kept over the
                // loop they would cost registers that Q and S need
                int ln = lane;
                asm volatile("" : "+v"(ln));
                // the next block's pieces; only copies issued after them are left.
                // Waves g and g + 4 share a SIMD: one does this first in a step and
                // the other last, so that the conversion, S, softmax and P.V of one
                // meet the S, softmax, P.V and conversion of its partner
                const auto next_tile = [&] {
                    if (!q8 || b + 1 >= n_raw) return;
                    if (b + 3 < n_raw)
                        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
                    else if (b + 2 < n_raw)
                        asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
                    else if (n_raw < b1)
                        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
                    else
                        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    convert(b + 1, ln);
                };
                int late = rg;  // (kept from becoming two copies of the loop)
                asm volatile("" : "+s"(late));
                if (late == 1) next_tile();
                const uint32_t k0 = tile_of(b), v0 = k0 + kTileV;
                const int r32 = ln & 31, hf = ln >> 5;
                // K fragment ks: row r32, chunk 2 ks + hf, its low 4 bits swizzled
                const uint32_t krow = k0 + r32 * 512 + 16 * (hf ^ p8_kswz(r32));
                f32x16 st;
                {
                    bf16x8_t kf[4];
                    const auto read = [&](int ks) { return as_bf16x8(lds_load16(krow ^ (32 * (ks & 7)), 256 * (ks >> 3))); };
#pragma unroll
                    for (int ks = 0; ks < 4; ks++) kf[ks] = read(ks);
                    constexpr f32x16 zero = {};
#pragma unroll
                    for (int ks = 0; ks < 16; ks++) {
                        const bf16x8_t ka = kf[ks & 3];
                        if (ks + 4 < 16) kf[ks & 3] = read(ks + 4);
                        st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka, qb[ks], ks ? st : zero, 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(kSgDsRead, 4, 0);
#pragma unroll
                    for (int ks = 0; ks < 16; ks++) {
                        if (ks + 4 < 16) __builtin_amdgcn_sched_group_barrier(kSgDsRead, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(kSgMfma, 1, 0);
                    }
                }
                // the next ids and scales: asked for here, where the LDS reads that
                // wait for scalar loads too are far
                ks_next = q8 ? scale_of(a.c.ks, b + 1, id[1]) : 1.f;
                vs_next = q8 ? scale_of(a.c.vs, b + 1, id[1]) : 1.f;
#pragma unroll
                for (int i = 0; i + 1 < kP8Raw; i++) id[i] = id[i + 1];
                id[kP8Raw - 1] = trow[min(b + kP8Raw, b1 - 1)];
                const float cq = c * kscale;  // >= 0 (or NaN)
                bf16x8_t pb[2], pl[2], pt[2];
                // lane: keys 8 (i / 4) + 4 hf + i % 4 of row r32.  A block
                // that the half's rows see whole keeps raw scores: the maximum is
                // scaled once and the scale enters the exponent through an FMA
                const auto softmax = [&] {
                    const bool full = b * kBlockTok + kBlockTok - 1 <= pos0 + row0 + 32 * rg && (b + 1) * kBlockTok <= kmax;
                    if (!full) {
                        asm volatile("");
                        const int qpos = min(pos0 + row0 + 32 * rg + r32, kmax - 1);
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            st[i] = b * kBlockTok + 8 * (i >> 2) + 4 * hf + (i & 3) <= qpos ? st[i] * cq : kNegBig;
                    }
                    const float cs = full ? cq : 1.f;
                    float mx = st[0];
#pragma unroll
                    for (int i = 1; i < 16; i++) mx = fmaxf(mx, st[i]);
                    mx = max_xor32(mx);
                    mx = full ? mx * cq : mx;
                    if (__builtin_amdgcn_ballot_w64(mx > m_run + kRescaleSlack) != 0) {
                        const bool up = mx > m_run + kRescaleSlack;
                        const float cr = up ? fast_exp2(m_run - mx) : 1.f;
                        m_run = up ? mx : m_run;
                        l_run *= cr;
#pragma unroll
                        for (int dt = 0; dt < 8; dt++) o[dt] *= cr;
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        u32x4 w, wl = {}, wt = {};
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            float y = fast_exp2(fmaf(st[8 * j + 2 * i], cs, -m_run));
                            float z = fast_exp2(fmaf(st[8 * j + 2 * i + 1], cs, -m_run));
                            l_run += y + z;
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
                        pb[j] = as_bf16x8(w);
                        pl[j] = as_bf16x8(wl);
                        pt[j] = as_bf16x8(wt);
                    }
                };
                const auto products = [&](auto&& read) {
                    bf16x8_t vf[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) vf[i] = read(i);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int dt = i & 7, j = i >> 3;  // products in a row are independent
                        const bf16x8_t va = vf[i & 3];
                        if (i + 4 < 16) vf[i & 3] = read(i + 4);
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pb[j], o[dt], 0, 0, 0);
                        if constexpr (FINE) {
                            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pl[j], o[dt], 0, 0, 0);
                            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pt[j], o[dt], 0, 0, 0);
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
                const auto pv = [&] {
                    if constexpr (q8) {
                        const uint32_t base = v0 + ln * 16;
                        products([&](int i) { return as_bf16x8(lds_load16(base, 2048 * (i & 7) + 1024 * (i >> 3))); });
                    } else {
                        // V^T through the transposing read: 16-lane group G takes dims
                        // 32 dt + 16 (G & 1) .. + 15 of rows 16 j + 4 hf + 0..3 (+ 8); its
                        // lane J addresses row J / 4, dims 4 (J % 4)
                        const int J = ln & 15, vr = 4 * hf + (J >> 2);
                        const uint32_t vtr = v0 + vr * 512 + 32 * ((ln >> 4) & 1) + 8 * (J & 3);
                        products([&](int i) {
                            // 64-B piece dt of rows vr (+ 8, + 16 j), all of one r & 7
                            const uint32_t y = vtr + (((i & 7) ^ (vr & 7)) << 6);
                            const u32x2 lo = lds_load_tr16(y, 8192 * (i >> 3)), hi = lds_load_tr16(y, 8192 * (i >> 3) + 4096);
                            return as_bf16x8(u32x4{lo[0], lo[1], hi[0], hi[1]});
                        });
                    }
                };
                softmax();
                pv();
                if (late == 0) next_tile();
            };
            int b = b0;
            for (; b < n_raw; b++) step(PfBuf<1>{}, b);
            for (; b < b1; b++) step(PfBuf<0>{}, b);
            const bool whole = b0 == 0 && b1 == it.n;
            const int part_slot = 2 * wg + (at > u_begin);
            {
                l_run = sum_xor32(l_run);
                if (32 * rg >= rows) {  // no rows
                } else if (!whole) {  // a part of the item's keys
                    float* part = a.part + (size_t)part_slot * kP8PartFloats;
                    float* acc = part + ((size_t)(2 * g + rg) * 32 * 64 + lane) * 4;
#pragma unroll
                    for (int dt = 0; dt < 8; dt++)
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            *reinterpret_cast<f32x4*>(acc + (dt * 4 + q) * 256) =
                                f32x4{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]};
                    if (hf == 0)
                        *reinterpret_cast<float2*>(part + kP8PartAcc + ((2 * g + rg) * 32 + r32) * 2) =
                            make_float2(m_run, l_run);
                } else if (32 * rg + r32 < rows) {
                    const size_t orow =
                        (((size_t)s * a.n_q + row0 + 32 * rg + r32) * kQHeads + h * kGroup + g) * kHeadDim + 4 * hf;
                    // (one copy per kind of gate, with nothing decided inside: the code
                    // runs once, and its fetch is what it costs)
                    const float inv = __builtin_amdgcn_rcpf(l_run);
                    const auto finish = [&](auto kind_) {
                        constexpr int kind = decltype(kind_)::value;  // 0: no gate, 1: exact, 2: the reference's
                        // gate words 8 pieces ahead: the stores keep loads behind them
                        uint2 gw[2][8];
                        const auto ask = [&](int i) {
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                gw[(i >> 3) & 1][k] = *reinterpret_cast<const uint2*>(a.gate + orow + 8 * (i + k));
                            asm volatile("" ::: "memory");
                        };
                        if constexpr (kind != 0) ask(0);
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            if constexpr (kind != 0)
                                if (i % 8 == 0 && i < 24) ask(i + 8);
                            const f32x16 y = o[i >> 2];
                            float f[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) f[k] = y[4 * (i & 3) + k] * inv;
                            if constexpr (kind != 0) {
                                float gs[4];
                                gate_factors(gw[(i >> 3) & 1][i & 7], kind == 2, gs);
#pragma unroll
                                for (int k = 0; k < 4; k++) f[k] *= gs[k];
                            }
                            if constexpr (FINE)
                                *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + orow + 8 * i) =
                                    f32x4{f[0], f[1], f[2], f[3]};
                            else
                                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + orow + 8 * i) =
                                    make_uint2(cvt_pk_bf16(f[0], f[1]), cvt_pk_bf16(f[2], f[3]));
                        }
                    };
                    if (!a.gate)
                        finish(PfBuf<0>{});
                    else if (a.gate_ref)
                        finish(PfBuf<2>{});
                    else
                        finish(PfBuf<1>{});
                }
            }
        }
        at = it.begin + b1;
    }
}

// Folds the partials of an item that the line's cuts went through: out =
// sum(w_p acc_p) / sum(w_p l_p), w_p = 2^(m_p - max m).  a.fold workgroups per
// cut (those of a cut that is not its item's first have nothing to do); a wave
// takes 32 rows of a q head x 32 dims at a time, as the parts stored them.
// Bound by the partials' bytes (262 KB each): 21 us after 16 sequences of 128
// rows over 256..6000 keys.
constexpr int kP8Fold = 3;  // parts requested at once
__global__ __launch_bounds__(256) void prefill_q8_combine_kernel(PrefillQ8Args a) {
    const int cut = blockIdx.x / a.fold + 1;  // between workgroups cut - 1 and cut
    const int u = a.cut[cut];
    const P8Item it = p8_find(a, a.seq_at[cut], u);
    // the cut is the item's first inner one (u = it.begin: no part before it)
    if (it.begin >= u || it.begin < a.cut[cut - 1]) return;
    const int lane = threadIdx.x & 63, r32 = lane & 31, hf = lane >> 5;
    const int row0 = it.rb * kP8Rows, rows = min(kP8Rows, a.n_q - row0);
    const int w0 = cut - 1;  // workgroups w0 .. w1 have a part of it
    int w1 = cut;
    while (a.cut[w1 + 1] < it.begin + it.n) w1++;
    // the first has it as its last run, unless its runs begin with it
    const int slot0 = 2 * w0 + (it.begin > a.cut[w0] ? 1 : 0);
    const auto slot = [&](int w) { return w == w0 ? slot0 : 2 * w; };
    for (int unit = (blockIdx.x % a.fold) * 4 + (threadIdx.x >> 6); unit < 64; unit += a.fold * 4) {
        const int row_group = unit >> 3, dt = unit & 7;  // (q head, half), dim tile
        const int rl = 32 * (row_group & 1) + r32;
        if (32 * (row_group & 1) >= rows) continue;
        const size_t orow =
            (((size_t)it.s * a.n_q + row0 + min(rl, rows - 1)) * kQHeads + it.h * kGroup + (row_group >> 1)) * kHeadDim +
            32 * dt + 4 * hf;
        uint2 gw[4];
#pragma unroll
        for (int q = 0; q < 4; q++)
            gw[q] = a.gate ? *reinterpret_cast<const uint2*>(a.gate + orow + 8 * q) : make_uint2(0u, 0u);
        float m = kNegBig, l = 0.f;
        f32x4 A[4] = {};
        for (int w = w0; w <= w1; w += kP8Fold) {
            float2 st[kP8Fold];
            f32x4 x[kP8Fold][4];
#pragma unroll
            for (int k = 0; k < kP8Fold; k++) {  // past the end: the last part again, not used
                const float* part = a.part + (size_t)slot(min(w + k, w1)) * kP8PartFloats;
                st[k] = *reinterpret_cast<const float2*>(part + kP8PartAcc + (row_group * 32 + r32) * 2);
#pragma unroll
                for (int q = 0; q < 4; q++)
                    x[k][q] = *reinterpret_cast<const f32x4*>(part + ((size_t)(row_group * 32 + dt * 4 + q) * 64 + lane) * 4);
            }
            float mx = m;
#pragma unroll
            for (int k = 0; k < kP8Fold; k++) mx = fmaxf(mx, st[k].x);
            const float cr = fast_exp2(m - mx);
            m = mx;
            l *= cr;
#pragma unroll
            for (int q = 0; q < 4; q++) A[q] *= cr;
#pragma unroll
            for (int k = 0; k < kP8Fold; k++) {
                if (w + k <= w1) {
                    const float wt = fast_exp2(st[k].x - m);
                    l = fmaf(wt, st[k].y, l);
#pragma unroll
                    for (int q = 0; q < 4; q++) A[q] += x[k][q] * wt;
                }
            }
        }
        if (rl >= rows) continue;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            float gs[4] = {1.f, 1.f, 1.f, 1.f};
            if (a.gate) gate_factors(gw[q], a.gate_ref, gs);
            const float o[4] = {A[q][0], A[q][1], A[q][2], A[q][3]};
            write_out(a.out, a.out_bf16, orow, 8 * q, a.gate != nullptr, gs, l, o);
        }
    }
}

int launch_prefill_q8(const PrefillQ8Args& a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const int grid = a.per_xcd * 8;
    if (a.out_bf16)
        hipLaunchKernelGGL(prefill_q8_kernel<false>, dim3(grid), dim3(512), 0, st, a);
    else
        hipLaunchKernelGGL(prefill_q8_kernel<true>, dim3(grid), dim3(512), 0, st, a);
    if (a.n_wgs > 1) hipLaunchKernelGGL(prefill_q8_combine_kernel, dim3((a.n_wgs - 1) * a.fold), dim3(256), 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace kvc
