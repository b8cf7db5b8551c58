// kvc_shared_kernels.h -- decode attention for sequences that share blocks, each
// shared block read once (included by kvc_kernels.hip).
//
// For every trie node (kvc_shared_plan.h) and kv head, the members' query rows
// (4 q heads each) attend to the node's keys in one product:
//   S^T[32 keys x 16 rows]  = K[keys x 256] . Q^T        (v_mfma_f32_16x16x32_bf16)
//   P^T = 2^(S^T - m), m the running maximum of the row
//   O^T[256 x 16 rows]     += V^T[256 x keys] . P^T
// in the operand layouts of the prefill kernel: a lane stays on one row in both
// products, P^T leaves the accumulator in operand order, and V^T fragments come
// from LDS through the transposing read.  A second launch folds the partials
// (m, l, O) of a row: O = sum 2^(m_p - M) O_p, l likewise, and divides.
#pragma once

namespace kvc {

struct SharedSmem {
    // kSharedRows: 4 stages of (K, V) units; otherwise (K, V) of each wave.
    // Rows of 512 B, 16-B chunks swizzled by the row (kswz, vswz).
    uint16_t unit[8][kBlockTok * kHeadDim];
    float2 ml[kWaves][16];
};
constexpr int kSharedStages = 4;
constexpr uint32_t kUnitLds = kBlockTok * kHeadDim * 2;
constexpr int kSharedRowPad = kHeadDim + 4;  // floats between rows of a wave's O in LDS
static_assert(16 * kSharedRowPad * 4 <= 2 * kUnitLds, "a wave's O fits its two units");

template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// PARTS: bf16 parts of a weight (1 for bf16 output, 3 = 24 bits for fp32 output)
template <int PARTS>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void shared_decode_kernel(SharedArgs a) {
    __shared__ SharedSmem sm;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q4 = lane >> 4, r16 = lane & 15;
    const int item = blockIdx.x;
    int node;
    {
        const int e0 = lane < a.n_nodes ? a.item_begin[lane + 1] : INT32_MAX;
        const int e1 = lane + 64 < a.n_nodes ? a.item_begin[lane + 65] : INT32_MAX;
        node = __popcll(__builtin_amdgcn_ballot_w64(e0 <= item)) + __popcll(__builtin_amdgcn_ballot_w64(e1 <= item));
        node = __builtin_amdgcn_readfirstlane(node);
    }
    if (node >= a.n_nodes) return;
    const SharedNode nd = a.node[node];
    const SharedShape sh = shared_shape(nd.shape);
    const int kind = sh.kind, chunk = sh.chunk, mb = sh.member_begin, members = sh.members;
    const int n_chunks = (nd.len + chunk - 1) / chunk;
    const int j = item - a.item_begin[node];
    int unit = j, grp = 0;
    if (members > kSharedSeqs) {
        // the groups of 16 members that read the same keys run on one XCD (b % 8), one after the other
        const int groups = (members + kSharedSeqs - 1) / kSharedSeqs;
        grp = (j >> 3) % groups;
        unit = (j >> 3) / groups * 8 + (j & 7);
        if (unit >= n_chunks * kKvHeads) return;
    }
    if (kind == kSharedHeads ? unit >= n_chunks : unit >= n_chunks * kKvHeads) return;  // (padding items)
    const int h = kind == kSharedHeads ? wave : unit % kKvHeads;
    const int ck = kind == kSharedHeads ? unit : unit / kKvHeads;
    const int b0 = ck * chunk, n_blk = min(chunk, nd.len - b0);
    const int s0 = __builtin_amdgcn_readfirstlane(a.member[mb]);
    const int32_t* trow = a.table + (size_t)a.slot[s0] * a.table_stride + nd.first + b0;

    // block ids: lane i holds this wave's i-th block
    const int step = kind == kSharedKeys ? kWaves : 1, base = kind == kSharedKeys ? wave : 0;
    const int n_my = (n_blk - base + step - 1) / step;
    const int idv = lane < n_my ? trow[base + lane * step] : 0;

    // this lane's row: member and q head
    const bool rows_kind = kind == kSharedRows;
    const int jm = rows_kind ? kSharedSeqs * grp + r16 : r16 >> 2;
    const int g = rows_kind ? wave : r16 & 3;
    const bool real = jm < members;
    const float c = fabsf(a.scale_log2);
    const uint32_t qflip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    bf16x8_t qb[8];
    {
        const int s = a.member[mb + min(jm, members - 1)];
        const uint16_t* qr = a.q + ((size_t)s * kQHeads + h * kGroup + g) * kHeadDim;
        u32x4 x[8];
#pragma unroll
        for (int ks = 0; ks < 8; ks++) x[ks] = *reinterpret_cast<const u32x4*>(qr + 32 * ks + 8 * q4);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
#pragma unroll
            for (int i = 0; i < 4; i++) x[ks][i] ^= qflip;
            // (waited for here, before the copies are issued: a later wait would cover those too)
            asm volatile("" : "+v"(x[ks]));
            qb[ks] = as_bf16x8(x[ks]);
        }
    }
    // keys of the chunk that exist (a node of one member may end inside a block)
    const int limit = members == 1 ? a.keys[s0] - (nd.first + b0) * kBlockTok : INT32_MAX;

    // copy instruction p of a unit: rows 2p, 2p + 1; lane l fills position l % 32
    const uint32_t cbk = (((lane & 31) ^ (lane >> 5)) << 4) + (lane >> 5) * 512;
    const uint32_t cbv = (((lane & 31) ^ ((lane >> 5) << 1)) << 4) + (lane >> 5) * 512;
    auto copy = [&](const uint16_t* pool, uint32_t cb, int jsh, int id, uint32_t lds, auto p0, auto np) {
        const uint16_t* src = pool + ((size_t)id * kKvHeads + h) * (kBlockTok * kHeadDim);
#pragma unroll
        for (int p = 0; p < decltype(np)::value; p++) {
            const int pp = p0 + p;
            lds_dma16s(src + pp * 2 * kHeadDim, cb ^ ((uint32_t)(pp & 7) << jsh), lds + pp * 1024);
        }
    };
    const uint32_t lds0 = lds_addr(&sm.unit[0][0]);

    f32x4 o[16], ol = {0.f, 0.f, 0.f, 0.f};  // ol: the row's sum of weights (PARTS 3: ol[0] is the lane's part)
    float m_run = kNegBig;
#pragma unroll
    for (int dt = 0; dt < 16; dt++) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    const bf16x8_t ones = as_bf16x8(u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});

    // operand fragments within a unit: K (kt, ks = 4 hi + jj): ka[jj] + 256 hi + 8192 kt;
    // V^T (dt, lo/hi): va[dt] + 8192 (hi)
    uint32_t ka[4], va[16];
#pragma unroll
    for (int jj = 0; jj < 4; jj++) ka[jj] = r16 * 512 + 16 * ((4 * jj + q4) ^ r16);
    {
        const int w = 4 * q4 + (r16 >> 2);
#pragma unroll
        for (int dt = 0; dt < 16; dt++) va[dt] = w * 512 + 16 * (2 * (dt ^ w) + ((r16 & 3) >> 1)) + 8 * (r16 & 1);
    }

    f32x4 st[2];
    auto scores = [&](uint32_t ku) {
        bf16x8_t kf[kPfAhead];
        auto read = [&](int i) {
            const int ks = i >> 1, kt = i & 1;
            kf[i % kPfAhead] = as_bf16x8(lds_load16(ku + ka[ks & 3], 256 * (ks >> 2) + 8192 * kt));
        };
#pragma unroll
        for (int i = 0; i < kPfAhead; i++) read(i);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int ks = i >> 1, kt = i & 1;
            const bf16x8_t x = kf[i % kPfAhead];
            if (i + kPfAhead < 16) read(i + kPfAhead);
            st[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, qb[ks], ks == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : st[kt], 0, 0, 0);
        }
    };
    bf16x8_t pw[PARTS];
    // weights of a block's scores; its keys from `valid` on do not exist
    auto weights = [&](int valid) {
        const bool all = valid >= kBlockTok;
        float cs = c;
        if (!all) {
            asm volatile("");
            cs = 1.f;
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int i = 0; i < 4; i++) st[kt][i] = 16 * kt + 4 * q4 + i < valid ? st[kt][i] * c : kNegBig;
        }
        float mx = kNegBig;
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int i = 0; i < 4; i++) mx = fmaxf(mx, st[kt][i]);
        mx = max_xor32(max_xor16(mx));
        const float mt = mx * cs;
        const bool up = mt > m_run + kRescaleSlack;
        if (__builtin_amdgcn_ballot_w64(up) != 0) {  // uniform; rows that keep their maximum scale by 1
            const float cr = up ? fast_exp2(m_run - mt) : 1.f;
            m_run = up ? mt : m_run;
#pragma unroll
            for (int dt = 0; dt < 16; dt++) o[dt] *= cr;
            ol *= cr;
        }
        const float nm = -m_run;
        u32x4 w[PARTS];
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float x = fast_exp2(fmaf(st[kt][2 * i], cs, nm)), y = fast_exp2(fmaf(st[kt][2 * i + 1], cs, nm));
                w[0][2 * kt + i] = cvt_pk_bf16(x, y);
                if constexpr (PARTS == 3) {
                    ol[0] += x + y;
                    const float x1 = x - bf16lo(w[0][2 * kt + i]), y1 = y - bf16hi(w[0][2 * kt + i]);  // exact
                    w[1][2 * kt + i] = cvt_pk_bf16(x1, y1);
                    w[2][2 * kt + i] = cvt_pk_bf16(x1 - bf16lo(w[1][2 * kt + i]), y1 - bf16hi(w[1][2 * kt + i]));
                }
            }
#pragma unroll
        for (int i = 0; i < PARTS; i++) pw[i] = as_bf16x8(w[i]);
    };
    auto values = [&](uint32_t vu) {
        bf16x8_t vf[kPfAhead];
        auto read = [&](int dt) {
            const u32x2 lo = lds_load_tr16(vu + va[dt], 0), hi = lds_load_tr16(vu + va[dt], 8192);
            vf[dt % kPfAhead] = as_bf16x8(u32x4{lo[0], lo[1], hi[0], hi[1]});
        };
#pragma unroll
        for (int i = 0; i < kPfAhead; i++) read(i);
#pragma unroll
        for (int dt = 0; dt < 16; dt++) {
            const bf16x8_t x = vf[dt % kPfAhead];
            if (dt + kPfAhead < 16) read(dt + kPfAhead);
#pragma unroll
            for (int i = 0; i < PARTS; i++) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, pw[i], o[dt], 0, 0, 0);
        }
        if constexpr (PARTS == 1) ol = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pw[0], ol, 0, 0, 0);
    };

    if (rows_kind) {
        // K and V of a block, for all waves; each copies an eighth of the rows.
        // 3 blocks are in flight while one is computed, one barrier a block.
        auto issue = [&](int i) {
            const int id = __builtin_amdgcn_readlane(idv, i);
            const uint32_t lds = lds0 + 2 * (i % kSharedStages) * kUnitLds;
            copy(a.kpool, cbk, 5, id, lds, 4 * wave, PfBuf<4>{});
            copy(a.vpool, cbv, 6, id, lds + kUnitLds, 4 * wave, PfBuf<4>{});
        };
        for (int i = 0; i < min(n_blk, kSharedStages - 1); i++) issue(i);
        for (int i = 0; i < n_blk; i++) {
            const int ahead = n_blk - 1 - i;  // uniform
            if (ahead >= 2)
                wait_vm<16>();
            else if (ahead == 1)
                wait_vm<8>();
            else
                wait_vm<0>();
            lds_barrier();  // block i is there, and every wave has read block i - 1
            if (i + kSharedStages - 1 < n_blk) issue(i + kSharedStages - 1);
            const uint32_t lds = lds0 + 2 * (i % kSharedStages) * kUnitLds;
            scores(lds);
            weights(kBlockTok);
            values(lds + kUnitLds);
        }
    } else {
        // a block of its own per wave: no barrier.  K of the next block is
        // requested once this one's has been read, V likewise.
        const uint32_t ku = lds0 + 2 * wave * kUnitLds, vu = ku + kUnitLds;
        auto issue = [&](const uint16_t* pool, uint32_t cb, int jsh, int i, uint32_t lds) {
            copy(pool, cb, jsh, __builtin_amdgcn_readlane(idv, i), lds, 0, PfBuf<16>{});
        };
        if (n_my > 0) {
            issue(a.kpool, cbk, 5, 0, ku);
            issue(a.vpool, cbv, 6, 0, vu);
        }
        for (int i = 0; i < n_my; i++) {
            const bool more = i + 1 < n_my;
            const int valid = limit - (base + i * step) * kBlockTok;
            wait_vm<16>();  // K: the 16 copies after it are V's
            scores(ku);
            wait_lds();
            if (more) issue(a.kpool, cbk, 5, i + 1, ku);
            weights(valid);
            if (more)
                wait_vm<16>();
            else
                wait_vm<0>();
            if (valid < kBlockTok) {  // rows that do not exist may hold anything: 0 times it must be 0
                for (int r = max(valid, 0); r < kBlockTok; r++)
                    *reinterpret_cast<u32x2*>(&sm.unit[2 * wave + 1][r * kHeadDim + lane * 4]) = u32x2{0u, 0u};
                wait_lds();
            }
            values(vu);
            wait_lds();
            if (more) issue(a.vpool, cbv, 6, i + 1, vu);
        }
    }
    float l = ol[0];
    if constexpr (PARTS == 3) l = sum_xor32(sum_xor16(l));

    const size_t row0 = (size_t)nd.row_begin + (size_t)(ck * kKvHeads + h) * members * kGroup;
    if (kind != kSharedKeys) {
        if (!real) return;
        const size_t row = row0 + jm * kGroup + g;
        float* acc = a.acc + row * kHeadDim + 4 * q4;
#pragma unroll
        for (int dt = 0; dt < 16; dt++) *reinterpret_cast<f32x4*>(acc + 16 * dt) = o[dt];
        if (q4 == 0) *reinterpret_cast<float2*>(a.stats + row * 2) = make_float2(m_run, l);
        return;
    }
    // fold the 4 waves' keys: O through LDS (each wave into its own units, which it alone read)
    float* own = reinterpret_cast<float*>(sm.unit[2 * wave]);
#pragma unroll
    for (int dt = 0; dt < 16; dt++) *reinterpret_cast<f32x4*>(own + r16 * kSharedRowPad + 16 * dt + 4 * q4) = o[dt];
    if (q4 == 0) sm.ml[wave][r16] = make_float2(m_run, l);
    __syncthreads();
    for (int r = wave; r < members * kGroup; r += kWaves) {
        float2 ml[kWaves];
        float m = kNegBig, lt = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            ml[w] = sm.ml[w][r];
            m = fmaxf(m, ml[w].x);
        }
        f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float f = fast_exp2(ml[w].x - m);
            lt = fmaf(f, ml[w].y, lt);
            t += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(sm.unit[2 * w]) + r * kSharedRowPad + lane * 4);
        }
        *reinterpret_cast<f32x4*>(a.acc + (row0 + r) * kHeadDim + lane * 4) = t;
        if (lane == 0) *reinterpret_cast<float2*>(a.stats + (row0 + r) * 2) = make_float2(m, lt);
    }
}

// One workgroup folds a (sequence, q head): each wave every 4th partial, its
// first kSharedFold requested before the weights are known.  The new token is
// a partial of its own, (score, 1, v), and is written to the cache.
constexpr int kSharedFold = 16;
__global__ __launch_bounds__(256) void shared_fold_kernel(SharedFoldArgs a) {
    __shared__ int rows[kSharedPath];
    __shared__ float wgt[kSharedPath];
    __shared__ float red[kWaves][2];
    __shared__ f32x4 part[kWaves][64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int s = blockIdx.x / kQHeads, head = blockIdx.x % kQHeads, h = head / kGroup, g = head % kGroup;
    int np = 0;
    for (int e = a.path_begin[s]; e < a.path_begin[s + 1]; e++) {
        const int pe = __builtin_amdgcn_readfirstlane(a.path[e]), node = pe & 255;
        const int nc = a.chunks[node] & 0xFFFF, mg = (a.chunks[node] >> 16) * kGroup;
        const int row = a.row_begin[node] + h * mg + (pe >> 8) * kGroup + g;
        for (int k = tid; k < nc; k += 256) rows[np + k] = row + k * kKvHeads * mg;
        np += nc;
    }
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
    __syncthreads();
    f32x4 x[kSharedFold];
    if (np > 0) {
#pragma unroll
        for (int k = 0; k < kSharedFold; k++)
            x[k] = *reinterpret_cast<const f32x4*>(a.acc + (size_t)rows[min(wave + kWaves * k, np - 1)] * kHeadDim + lane * 4);
    }
    float ms[kSharedPath / 256], ls[kSharedPath / 256], m = kNegBig;
#pragma unroll
    for (int i = 0; i < kSharedPath / 256; i++) {
        ms[i] = kNegBig;
        ls[i] = 0.f;
        if (tid + 256 * i < np) {
            const float2 t = *reinterpret_cast<const float2*>(a.stats + (size_t)rows[tid + 256 * i] * 2);
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
        t += wgt[p] * *reinterpret_cast<const f32x4*>(a.acc + (size_t)rows[p] * kHeadDim + lane * 4);
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
            const int pos = a.keys[s];
            const int blk = a.table[(size_t)a.slot[s] * a.table_stride + pos / kBlockTok];
            const size_t off = (((size_t)blk * kKvHeads + h) * kBlockTok + pos % kBlockTok) * kHeadDim + lane * 4;
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
    hipLaunchKernelGGL(shared_fold_kernel, dim3(f.n_seqs * kQHeads), dim3(256), 0, st, f);
    return (int)hipGetLastError();
}

}  // namespace kvc
