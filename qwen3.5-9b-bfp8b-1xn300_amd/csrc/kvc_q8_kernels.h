// kvc_q8_kernels.h -- kernels of the 8-bit K/V blocks: quantize, gather, and
// decode attention over sequences that start with 8-bit blocks.  Included by
// kvc_kernels.hip, whose helpers it uses.
//
// A unit (32 tokens of one kv head, K or V) holds x = i s, i int8, s fp32;
// its pieces lie in matrix-operand order (kvc_internal.h).
#pragma once

namespace kvc {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float nan_f() { return __uint_as_float(0x7FC00000u); }

// First s with begin[s + 1] > i.
__device__ __forceinline__ int find_seq(const int32_t* begin, int n, int i) {
    int s = 0;
    while (s + 1 < n && begin[s + 1] <= i) s++;
    return s;
}

// Offset of byte (token, dim) in a K or V unit.
__device__ __forceinline__ int q8_k_off(int tok, int d) {
    return (((tok >> 4) * 4 + (d >> 6)) * 64 + ((d >> 4) & 3) * 16 + (tok & 15)) * 16 + (d & 15);
}
__device__ __forceinline__ int q8_v_off(int tok, int d) {
    const int g = ((tok >> 2) & 1) + 2 * (tok >> 4), e = (tok & 3) + 4 * ((tok >> 3) & 1);
    return ((d >> 5) * 64 + g * 16 + (d & 15)) * 16 + ((d >> 4) & 1) * 8 + e;
}

// ---------------------------------------------------------------------------
// Quantize: one workgroup = one unit.  s = max(a, 2^-100) / 127 and
// i = rne(x * (127 / max(a, 2^-100))) with a = max |x|; the product's own
// rounding (2^-24 of 127) can carry an element over a tie, nothing else.  The
// floor under a keeps the reciprocal finite: a unit of smaller values reads as
// (nearly) zeros.  A unit with an infinity or a NaN gets s = NaN, so that
// everything computed from it is NaN, as it would be from the bf16 rows.
// V pieces hold 8 tokens of a dim, so the unit is turned through LDS.  Bound by
// memory: each byte is read once and the unit sits in registers between the
// maximum and the rounding.  8 layers of 4096 tokens (134 MB read, 67 written)
// 36 us, 5.6 TB/s; 2 layers of 16 x 992 tokens 32 us, 6.1 TB/s.
__global__ __launch_bounds__(256) void quantize_kernel(QuantizeArgs a) {
    __shared__ __align__(16) uint16_t tile[kBlockTok * kHeadDim];
    __shared__ uint32_t wmax[4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int per = a.p.n_layers * 2 * kKvHeads;
    const int i = blockIdx.x / per, u = blockIdx.x % per;
    const int h = u % kKvHeads, kv = (u / kKvHeads) & 1, lkv = u / kKvHeads;
    const int s = find_seq(a.begin, a.n_seqs, i);
    const int b = a.first[s] + i - a.begin[s];
    const int id = a.p.table[(size_t)a.src[s] * a.p.table_stride + b];
    const int id8 = a.p.table[(size_t)a.dst[s] * a.p.table_stride + b];
    const u32x4* src = reinterpret_cast<const u32x4*>(a.p.pool + (int64_t)lkv * a.p.layer_kv_bytes +
                                                      ((size_t)id * kKvHeads + h) * kUnitBytes);
    u32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = __builtin_nontemporal_load(src + j * 256 + t);
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            mx = max(mx, x[j][k] & 0x7FFFu);
            mx = max(mx, (x[j][k] >> 16) & 0x7FFFu);
        }
    // largest magnitude, as bf16 bits (ordered as integers, NaN above infinity)
    mx = (uint32_t)wave_max((float)mx);
    if (lane == 0) wmax[wave] = mx;
#pragma unroll
    for (int j = 0; j < 4; j++) reinterpret_cast<u32x4*>(tile)[j * 256 + t] = x[j];
    __syncthreads();
    mx = max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3]));
    const bool bad = mx >= 0x7F80u;
    const float amax = fmaxf(__uint_as_float(mx << 16), 0x1p-100f);
    const float scale = bad ? nan_f() : amax / 127.0f, inv = bad ? 0.f : 127.0f / amax;
    const auto q1 = [&](uint16_t w) -> uint32_t {
        const float y = __builtin_amdgcn_fmed3f(rintf(bf16f(w) * inv), -127.f, 127.f);
        return (uint32_t)(int)(bad ? 0.f : y) & 0xFFu;
    };
    u32x4* out = reinterpret_cast<u32x4*>(a.p.q8 + (int64_t)lkv * a.p.q8_kv_bytes +
                                          ((size_t)id8 * kKvHeads + h) * kQ8UnitBytes);
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int e = j * 4 + wave;  // piece group: 64 pieces
        u32x4 o;
        if (kv == 0) {
            const uint16_t* row = tile + (16 * (e >> 2) + c) * kHeadDim + 64 * (e & 3) + 16 * g;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint2 w = reinterpret_cast<const uint2*>(row)[k];
                o[k] = q1(w.x & 0xFFFF) | q1(w.x >> 16) << 8 | q1(w.y & 0xFFFF) << 16 | q1(w.y >> 16) << 24;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint16_t* col =
                    tile + (16 * (g >> 1) + 4 * (g & 1) + 8 * (k & 1)) * kHeadDim + 32 * e + 16 * (k >> 1) + c;
                o[k] = q1(col[0]) | q1(col[kHeadDim]) << 8 | q1(col[2 * kHeadDim]) << 16 | q1(col[3 * kHeadDim]) << 24;
            }
        }
        __builtin_nontemporal_store(o, out + e * 64 + lane);
    }
    if (t == 0) a.p.scales[(int64_t)lkv * a.p.scale_kv + (int64_t)id8 * kKvHeads + h] = scale;
}

// ---------------------------------------------------------------------------
// Gather over sequences with 8-bit blocks: one workgroup = one unit of a cache
// block that the range [tok0, tok0 + n) of its sequence touches.  8-bit units
// become bf16(i s) rows in LDS first, so that the output rows (512 B a token
// and head) are written whole.  One layer of 16 x 1000 tokens 20 us, 4.9 TB/s;
// of 4096 tokens 6.5 us, of which most is the launch and one memory latency.
__global__ __launch_bounds__(256) void gather_q8_kernel(GatherQ8Args a) {
    // rows 16 B apart from a multiple of 128 B: 16 lanes that write one dim
    // range of 16 tokens fall on different banks
    constexpr int kRow = kHeadDim + 8;
    __shared__ __align__(16) uint16_t tile[kBlockTok * kRow];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int item = blockIdx.x >> 3, h = blockIdx.x & 3, kv = (blockIdx.x >> 2) & 1;
    const int s = find_seq(a.item_begin, a.n_seqs, item);
    const int b = a.tok0 / kBlockTok + item - a.item_begin[s];
    const int nt = a.out_begin[s + 1] - a.out_begin[s];
    const int p0 = max(a.tok0, b * kBlockTok), p1 = min(a.tok0 + nt, (b + 1) * kBlockTok);
    const int id = a.c.table[(size_t)a.slot[s] * a.c.table_stride + b];
    uint16_t* out = (kv ? a.v_out : a.k_out) + (size_t)a.out_begin[s] * kKvHeads * kHeadDim;
    const bool q8 = b < a.n8[s];
    if (q8) {
        const size_t unit = (size_t)id * kKvHeads + h;
        const u32x4* src = reinterpret_cast<const u32x4*>((kv ? a.c.v8 : a.c.k8) + unit * kQ8UnitBytes);
        const float scale = (kv ? a.c.vs : a.c.ks)[unit];
        const int c = lane & 15, g = lane >> 4;
        u32x4 x[2];
#pragma unroll
        for (int j = 0; j < 2; j++) x[j] = src[(j * 4 + wave) * 64 + lane];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int e = j * 4 + wave;
            uint32_t w[8];  // packed pairs in piece order
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int y = (int)x[j][k];
                w[2 * k] = cvt_pk_bf16((float)((y << 24) >> 24) * scale, (float)((y << 16) >> 24) * scale);
                w[2 * k + 1] = cvt_pk_bf16((float)((y << 8) >> 24) * scale, (float)(y >> 24) * scale);
            }
            if (kv == 0) {
                u32x4* dst = reinterpret_cast<u32x4*>(tile + (16 * (e >> 2) + c) * kRow + 64 * (e & 3) + 16 * g);
                dst[0] = u32x4{w[0], w[1], w[2], w[3]};
                dst[1] = u32x4{w[4], w[5], w[6], w[7]};
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) {  // tokens (2k, 2k + 1) % 4 of their groups
                    const int tok = 16 * (g >> 1) + 4 * (g & 1) + 8 * ((k >> 1) & 1) + 2 * (k & 1);
                    const int d = 32 * e + 16 * (k >> 2) + c;
                    tile[tok * kRow + d] = (uint16_t)w[k];
                    tile[(tok + 1) * kRow + d] = (uint16_t)(w[k] >> 16);
                }
            }
        }
        __syncthreads();
    }
    const uint16_t* from = (kv ? a.c.vpool : a.c.kpool) + ((size_t)id * kKvHeads + h) * kBlockTok * kHeadDim;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int tok = j * 8 + (t >> 5), part = t & 31, pos = b * kBlockTok + tok;
        if (pos < p0 || pos >= p1) continue;
        const u32x4 x = *reinterpret_cast<const u32x4*>(q8 ? tile + tok * kRow + part * 8 : from + tok * kHeadDim + part * 8);
        __builtin_nontemporal_store(
            x, reinterpret_cast<u32x4*>(out + ((size_t)(pos - a.tok0) * kKvHeads + h) * kHeadDim + part * 8));
    }
}

// ---------------------------------------------------------------------------
// Decode over 8-bit blocks.  A wave takes whole blocks of its chunk (one kv
// head), straight from memory into matrix operands, and works in int8
// products with int32 sums, which are exact:
//   q of a head = 2^(e - 29) (sum over k of 256^k Q_k), 2^e the power of two at
//     or below the row's largest value, Q_k signed base-256 digits; the 4 digit
//     planes of the 4 heads are the 16 rows of the A operand, K's tokens the
//     columns.  bf16 values from 2^(e - 22) on are exact in them.  If the wave
//     has smaller ones that are not, what is left of them, in 30 more bits, takes
//     4 more planes and a second set of products (they decide the scores where
//     K is near 0 in the large channels)
//   s = 2^(e - 29) scale ks (sum over k of 256^k Q_k . K)
//   p = 2^(s - m), m = the block's largest score of the head, in 30-bit digits
//     likewise; o += 2^(m - M) vs 2^-30 (sum over k of 256^k P_k . V)
// with fp32 running M (the offset, raised when a block exceeds it by the
// slack), sum and o.  Digits relative to the block's own maximum lose less
// than 2^-30 of it per weight, whatever other blocks hold.  The matrix pipe
// has rows to spare (4 heads of 16 rows), so the digits are free; the block's
// 16 KiB cost about 220 VALU instructions and 24 MFMAs.
// Bound by memory from some tens of sequences on: 64 sequences of 512..16384
// tokens 179 us, 1037 MB at 5.8 TB/s; 8 of 777..6001 21 us a layer, 3.4 TB/s
// (the run-up of 2 workgroups a CU); below that by latency: 1 x 4096 9.5 us, 1 x
// 300 7.5 us a layer (kernel trace; a layer of calls back to back 9.0 and 6.9).
// The second planes, with fp32 output: 64 sequences 180 us against 179, 1 x 4096
// as without.
//
// digits: bytes 0..3 of dig30(x) are x's signed base-256 digits
__device__ __forceinline__ uint32_t dig30(int n) { return ((uint32_t)n + 0x00808080u) ^ 0x00808080u; }

struct Q8Wave {
    i32x4_t q[4];      // A operand: row (plane k = c / 4, head c % 4), dims 64 s + 16 g .. +15
    bool low;          // the planes of what q leaves are in use (LDS, laid out as q's)
    float qs[2];       // 2^(e - 29) scale log2(e) of heads 2 (g / 2), + 1
    float acc[16][4];  // dims 16 t + c of head r, plane g's share
    float m[2], l[2];  // of heads 2 (g / 2), + 1: offset (uniform over the heads' lanes), lane's part of the sum
};

struct Q8Block {
    u32x4 k[8], v[8];
    float ks, vs;
};

__device__ __forceinline__ void q8_load(Q8Block& r, const MixedCache& c, int id, int h, int lane) {
    const size_t unit = (size_t)id * kKvHeads + h;
    const u32x4* k = reinterpret_cast<const u32x4*>(c.k8 + unit * kQ8UnitBytes) + lane;
    const u32x4* v = reinterpret_cast<const u32x4*>(c.v8 + unit * kQ8UnitBytes) + lane;
#pragma unroll
    for (int i = 0; i < 8; i++) r.k[i] = __builtin_nontemporal_load(k + 64 * i);
#pragma unroll
    for (int i = 0; i < 8; i++) r.v[i] = __builtin_nontemporal_load(v + 64 * i);
    r.ks = c.ks[unit];
    r.vs = c.vs[unit];
}

// q's digit planes.  Lane (g, c) digests dims 64 s + 16 g .. +15, s = c / 4, of
// head c % 4 and hands the 4 planes to the lanes that hold them as operand.
__device__ __forceinline__ void q8_load_q(Q8Wave& w, const uint16_t* qhead0, float scale_log2, u32x4* lds, int lane) {
    const int c = lane & 15, g = lane >> 4, head = c & 3, sp = c >> 2;
    const u32x4* src = reinterpret_cast<const u32x4*>(qhead0 + head * kHeadDim + 64 * sp + 16 * g);
    const u32x4 x0 = src[0], x1 = src[1];
    float f[16];
    // largest magnitude and, less one bit pattern, the smallest that is not 0, of
    // even and of odd elements (bf16 bits order as integers)
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 most = {0, 0}, least = {0xFFFF, 0xFFFF};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t w = i < 4 ? x0[i & 3] : x1[i & 3];
        f[2 * i] = bf16lo(w);
        f[2 * i + 1] = bf16hi(w);
        const u16x2 a = __builtin_bit_cast(u16x2, w & 0x7FFF7FFFu);
        most = __builtin_elementwise_max(most, a);
        least = __builtin_elementwise_min(least, a - u16x2{1, 1});
    }
    uint32_t mx = max((uint32_t)most[0], (uint32_t)most[1]);
    // the head's maximum over its 16 lanes (c / 4 and g); bits are exact in fp32
    float mf = (float)mx;
    mf = fmaxf(mf, dpp<kDppRowRor8>(mf));
    mf = fmaxf(mf, dpp<0x124>(mf));  // row rotate by 4
    mf = max_xor16(mf);
    mf = max_xor32(mf);
    mx = (uint32_t)mf;
    const uint32_t e = max(mx >> 7, 127u - 90u) << 23;  // 2^e as fp32 bits, at least 2^-90
    const bool bad = mx >= 0x7F80u;
    const float up = __uint_as_float(((2 * 127 + 29) << 23) - e);  // 2^(29 - e)
    // an element under 2^(e - 22) may have bits below the digits
    w.low = __builtin_amdgcn_ballot_w64(min((uint32_t)least[0], (uint32_t)least[1]) < (e >> 16) - (22u << 7)) != 0;
    uint32_t dg[16];
    const auto planes = [&] {
#pragma unroll
        for (int k = 0; k < 4; k++) {  // plane k: byte k of each digit word
            u32x4 o;
            const uint32_t sel = (uint32_t)k | (uint32_t)(k + 4) << 8 | 0x0C0C0000u;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t lo = __builtin_amdgcn_perm(dg[4 * i + 1], dg[4 * i], sel);
                const uint32_t hi = __builtin_amdgcn_perm(dg[4 * i + 3], dg[4 * i + 2], sel);
                o[i] = lo | hi << 16;
            }
            lds[((k * 4 + head) * 4 + sp) * 4 + g] = o;
        }
        wave_lds_sync();
    };
#pragma unroll
    for (int i = 0; i < 16; i++) {
        f[i] = bad ? 0.f : f[i] * up;  // exact
        dg[i] = dig30((int)f[i]);
    }
    planes();
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const u32x4 o = lds[(c * 4 + s) * 4 + g];
        w.q[s] = __builtin_bit_cast(i32x4_t, o);
    }
    if (w.low) {  // what the cut left, below 1 in magnitude
        wave_lds_sync();
#pragma unroll
        for (int i = 0; i < 16; i++) dg[i] = dig30((int)((f[i] - truncf(f[i])) * 0x1p30f));
        planes();
    }
    const float mine = bad ? nan_f() : __uint_as_float(e) * 0x1p-29f * scale_log2;
    const float h0 = readlane(mine, 0), h1 = readlane(mine, 1), h2 = readlane(mine, 2), h3 = readlane(mine, 3);
    w.qs[0] = g < 2 ? h0 : h2;
    w.qs[1] = g < 2 ? h1 : h3;
    wave_lds_sync();
}

__device__ __forceinline__ float swap16_add(float a, float b) {  // row 0: a's rows 0, 1; row 1: b's; rows 2, 3 likewise
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap32_add(float a, float b) {  // lower half: a's halves; upper half: b's
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ void q8_block(const Q8Block& b, Q8Wave& w, const u32x4* lds, uint32_t* pl, float w256, int lane) {
    const int c = lane & 15, g = lane >> 4;
    // planes x keys: lane holds plane g of heads r = 0..3, keys 16 t + c
    i32x4_t s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 4; s++) {
        s0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(w.q[s], __builtin_bit_cast(i32x4_t, b.k[s]), s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(w.q[s], __builtin_bit_cast(i32x4_t, b.k[4 + s]), s1, 0, 0, 0);
    }
    float y0[4], y1[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        y0[r] = (float)s0[r] * w256;
        y1[r] = (float)s1[r] * w256;
    }
    if (w.low) {
        s0 = s1 = i32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const u32x4 o = lds[(c * 4 + s) * 4 + g];
            s0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, o), __builtin_bit_cast(i32x4_t, b.k[s]), s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, o), __builtin_bit_cast(i32x4_t, b.k[4 + s]), s1, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            y0[r] = fmaf((float)s0[r], w256 * 0x1p-30f, y0[r]);
            y1[r] = fmaf((float)s1[r], w256 * 0x1p-30f, y1[r]);
        }
    }
    // sum of the planes; lane (g, c) ends with key 16 (g & 1) + c of heads
    // 2 (g / 2) and + 1
    float x[4];
#pragma unroll
    for (int r = 0; r < 4; r++) x[r] = swap16_add(y0[r], y1[r]);
    float sc[2], p[2], f[2];
    bool up = false;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        sc[j] = swap32_add(x[j], x[2 + j]) * (w.qs[j] * b.ks);
        float mx = sc[j];
        mx = fmaxf(mx, dpp<kDppXor1>(mx));
        mx = fmaxf(mx, dpp<kDppXor2>(mx));
        mx = fmaxf(mx, dpp<kDppHalfMirror>(mx));
        mx = fmaxf(mx, dpp<kDppRowRor8>(mx));
        mx = max_xor16(mx);
        p[j] = fast_exp2(sc[j] - mx);
        f[j] = mx;
        up |= mx > w.m[j] + kRescaleSlack;
    }
    if (__builtin_amdgcn_ballot_w64(up) != 0) {
        float cr[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const float mn = f[j] > w.m[j] + kRescaleSlack ? f[j] : w.m[j];
            cr[j] = fast_exp2(w.m[j] - mn);
            w.m[j] = mn;
            w.l[j] *= cr[j];
        }
        const float c0 = readlane(cr[0], 0), c1 = readlane(cr[1], 0), c2 = readlane(cr[0], 32), c3 = readlane(cr[1], 32);
#pragma unroll
        for (int t = 0; t < 16; t++) {
            w.acc[t][0] *= c0;
            w.acc[t][1] *= c1;
            w.acc[t][2] *= c2;
            w.acc[t][3] *= c3;
        }
    }
    // digits of p to LDS at [head][position of the key in V's token order]
    // (token 16 (g & 1) + c: group 2 (g & 1) + (c / 4) % 2, element c % 4 + 4 (c / 8))
    const int pos = 16 * (g & 1) + 8 * ((c >> 2) & 1) + (c & 3) + 4 * (c >> 3), h0 = 2 * (g >> 1);
#pragma unroll
    for (int j = 0; j < 2; j++) {
        f[j] = fast_exp2(f[j] - w.m[j]);
        w.l[j] = fmaf(p[j], f[j], w.l[j]);
        pl[(h0 + j) * kBlockTok + pos] = dig30((int)(p[j] * 0x1p30f));
    }
    // per head: 2^(m - M) vs 2^-30, and the lane's plane
    const float vf = b.vs * 0x1p-30f * w256;
    float F[4];
    F[0] = readlane(f[0], 0) * vf;
    F[1] = readlane(f[1], 0) * vf;
    F[2] = readlane(f[0], 32) * vf;
    F[3] = readlane(f[1], 32) * vf;
    wave_lds_sync();
    const u32x4* pr = reinterpret_cast<const u32x4*>(pl + (c & 3) * kBlockTok + 8 * g);
    const u32x4 d0 = pr[0], d1 = pr[1];
    const uint32_t k = (uint32_t)c >> 2, sel = k | (k + 4) << 8 | 0x0C0C0000u;
    const uint32_t a0 = __builtin_amdgcn_perm(d0[1], d0[0], sel) | __builtin_amdgcn_perm(d0[3], d0[2], sel) << 16;
    const uint32_t a1 = __builtin_amdgcn_perm(d1[1], d1[0], sel) | __builtin_amdgcn_perm(d1[3], d1[2], sel) << 16;
    const long pa = (long)((uint64_t)a0 | (uint64_t)a1 << 32);
    wave_lds_sync();
#pragma unroll
    for (int t = 0; t < 16; t++) {
        const u32x4 v = b.v[t >> 1];
        const long vb = (long)((uint64_t)v[2 * (t & 1)] | (uint64_t)v[2 * (t & 1) + 1] << 32);
        const i32x4_t o = __builtin_amdgcn_mfma_i32_16x16x32_i8(pa, vb, i32x4_t{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; r++) w.acc[t][r] = fmaf((float)o[r], F[r], w.acc[t][r]);
    }
}

struct DecodeQ8Smem {
    union {
        DecodeSmem d;
        struct {
            u32x4 q[kWaves][256];                         // q's digit planes, 4 KiB a wave
            uint32_t p[kWaves][kGroup * kBlockTok];       // p's digits
        } w;
    };
    __align__(16) uint16_t p16[kWaves][64];  // 32 floats a wave
};

__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void decode_q8_kernel(DecodeQ8Args a) {
    __shared__ DecodeQ8Smem sm;
    const int bid = blockIdx.x;
    const int item = (bid & 7) * a.per_xcd + (bid >> 3);
    if (item >= a.n_items) return;
    const int h = item / a.total_chunks;
    const int chunk = item - h * a.total_chunks;
    const int s = find_seq(a.chunk_begin, a.n_seqs, chunk);
    const int n_chunks = a.chunk_begin[s + 1] - a.chunk_begin[s];
    const int ci = chunk - a.chunk_begin[s];
    const int L = a.kv_len[s], n8 = a.n8[s];
    const int n_blocks = (L + kBlockTok - 1) / kBlockTok;
    const int chunks8 = (n8 + a.cb8 - 1) / a.cb8;
    const int32_t* trow = a.c.table + (size_t)a.slot[s] * a.c.table_stride;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint16_t* qhead0 = a.q + ((size_t)s * kQHeads + h * kGroup) * kHeadDim;
    float M, Lsum, A[4];
    if (ci < chunks8) {
        const int blk0 = ci * a.cb8, blk1 = min(blk0 + a.cb8, n8);
        Q8Wave w;
        Q8Block r0, r1;
        int b = blk0 + wave;
        // (a wave without a block loads the chunk's first and does not use it)
        q8_load(r0, a.c, trow[b < blk1 ? b : blk0], h, lane);
        q8_load_q(w, qhead0, a.scale_log2, sm.w.q[wave], lane);
#pragma unroll
        for (int t = 0; t < 16; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) w.acc[t][r] = 0.f;
        w.m[0] = w.m[1] = kNegBig;
        w.l[0] = w.l[1] = 0.f;
        const int g = lane >> 4, c = lane & 15;
        const float w256 = __uint_as_float((127u + 8u * g) << 23);  // 256^g
        uint32_t* pl = sm.w.p[wave];
        for (; b < blk1; b += 2 * kWaves) {
            if (b + kWaves < blk1) q8_load(r1, a.c, trow[b + kWaves], h, lane);
            q8_block(r0, w, sm.w.q[wave], pl, w256, lane);
            if (b + kWaves >= blk1) break;
            if (b + 2 * kWaves < blk1) q8_load(r0, a.c, trow[b + 2 * kWaves], h, lane);
            q8_block(r1, w, sm.w.q[wave], pl, w256, lane);
        }
        // sum the planes: lane (g, c) ends with dims 16 t + c of the 4 tiles
        // t = i + 4 (g / 2) + 8 (g & 1), i = 0..3
        float y[4][kGroup];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            float x[8];
#pragma unroll
            for (int t = 0; t < 8; t++) x[t] = swap16_add(w.acc[t][r], w.acc[t + 8][r]);
#pragma unroll
            for (int t = 0; t < 4; t++) y[t][r] = swap32_add(x[t], x[t + 4]);
        }
        float lt[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            float x = w.l[j];
            x += dpp<kDppXor1>(x);
            x += dpp<kDppXor2>(x);
            x += dpp<kDppHalfMirror>(x);
            x += dpp<kDppRowRor8>(x);
            lt[j] = sum_xor16(x);
        }
        __syncthreads();  // the digit areas give way to the merge's
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) sm.d.acc[wave][r][16 * (t + 4 * (g >> 1) + 8 * (g & 1)) + c] = y[t][r];
        if (c == 0 && (g & 1) == 0) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                sm.d.ml[wave][g + j][0] = w.m[j];
                sm.d.ml[wave][g + j][1] = lt[j];
            }
        }
        __syncthreads();
        const int gg = threadIdx.x >> 6, d0 = (threadIdx.x & 63) * 4;
        M = kNegBig;
#pragma unroll
        for (int v = 0; v < kWaves; v++) M = fmaxf(M, sm.d.ml[v][gg][0]);
        Lsum = 0.f;
        A[0] = A[1] = A[2] = A[3] = 0.f;
#pragma unroll
        for (int v = 0; v < kWaves; v++) {
            const float wt = fast_exp2(sm.d.ml[v][gg][0] - M);
            Lsum = fmaf(wt, sm.d.ml[v][gg][1], Lsum);
            const float4 x = *reinterpret_cast<const float4*>(&sm.d.acc[v][gg][d0]);
            A[0] = fmaf(wt, x.x, A[0]);
            A[1] = fmaf(wt, x.y, A[1]);
            A[2] = fmaf(wt, x.z, A[2]);
            A[3] = fmaf(wt, x.w, A[3]);
        }
    } else {
        // bf16 blocks: the bf16 decode's walk, with weights and P.V in fp32
        const int blk0 = n8 + (ci - chunks8) * a.cbf, blk1 = min(blk0 + a.cbf, n_blocks);
        const bool fused_new = a.k_new != nullptr;
        const int Lw = fused_new ? L - 1 : L;
        const int n_walk = max(0, min(blk1, (Lw + kBlockTok - 1) / kBlockTok) - blk0);
        const int first_ids = lane < min(64, blk1 - blk0) ? trow[blk0 + lane] : 0;
        uint32_t qv[kGroup][2][4];
        load_q(qv, qhead0, lane);
        WaveState st;
        init_state(st);
        walk_blocks<1, false, true>(a.c.kpool, a.c.vpool, trow, h, blk0, n_walk, Lw, qv, a.scale_log2, sm.p16[wave], st,
                                    wave, lane, 0, first_ids, [] {});
        finalize_l(st);
        if (fused_new && L - 1 >= blk0 * kBlockTok && L - 1 < blk1 * kBlockTok && wave == 0) {
            const uint16_t* knew = a.k_new + ((size_t)s * kKvHeads + h) * kHeadDim;
            const uint16_t* vnew = a.v_new + ((size_t)s * kKvHeads + h) * kHeadDim;
            fold_token<1>(st, qv, knew, vnew, a.scale_log2, lane, 0);
            append_new_token(const_cast<uint16_t*>(a.c.kpool), const_cast<uint16_t*>(a.c.vpool),
                             trow[(L - 1) / kBlockTok], h, L - 1,
                             *reinterpret_cast<const u32x4*>(((lane >> 5) ? vnew : knew) + (lane & 31) * 8));
        }
        merge_waves(st, sm.d, wave, lane, M, Lsum, A);
    }
    const int t = threadIdx.x, g = t >> 6, d0 = (t & 63) * 4;
    const size_t orow = ((size_t)s * kQHeads + h * kGroup + g) * kHeadDim;
    const bool has_gate = a.gate != nullptr;
    const uint2 gw = has_gate ? *reinterpret_cast<const uint2*>(a.gate + orow + d0) : make_uint2(0u, 0u);
    float gs[4] = {1.f, 1.f, 1.f, 1.f};
    if (n_chunks == 1) {
        if (has_gate) gate_factors(gw, a.gate_ref, gs);
        write_out(a.out, a.out_bf16, orow, d0, has_gate, gs, Lsum, A);
        return;
    }
    // split-K exchange: decode_kernel's, with its partials and counters
    const __amdgpu_buffer_rsrc_t prs = make_rsrc(a.part, a.part_bytes);
    const int ibase = item * kItemFloats * 4;
    const u32x4 av = {__float_as_uint(A[0]), __float_as_uint(A[1]), __float_as_uint(A[2]), __float_as_uint(A[3])};
    __builtin_amdgcn_raw_buffer_store_b128(av, prs, ibase + (g * kHeadDim + d0) * 4, 0, kCpolSC1);
    if (lane == 0) {
        const u32x2 mlv = {__float_as_uint(M), __float_as_uint(Lsum)};
        __builtin_amdgcn_raw_buffer_store_b64(mlv, prs, ibase + (kGroup * kHeadDim + 2 * g) * 4, 0, kCpolSC1);
    }
    __builtin_amdgcn_s_waitcnt(0);
    int32_t* ctr = a.counters + ((s * kKvHeads + h) * kMaxDParts * kGroup + g) * kCounterStride;
    int prev = 0;
    if (lane == 0) prev = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__builtin_amdgcn_readfirstlane(prev) != n_chunks - 1) return;
    asm volatile("" ::: "memory");
    float Mc = kNegBig, Lc = 0.f, Ac[4] = {0.f, 0.f, 0.f, 0.f};
    const int first = h * a.total_chunks + a.chunk_begin[s];
    for (int k0 = 0; k0 < n_chunks; k0 += kCombineBatch) {
        const int nk = min(kCombineBatch, n_chunks - k0);
        if (nk <= 8)
            combine_batch<8>(prs, first + k0, nk, g, d0, lane, Mc, Lc, Ac);
        else if (nk <= 16)
            combine_batch<16>(prs, first + k0, nk, g, d0, lane, Mc, Lc, Ac);
        else
            combine_batch<32>(prs, first + k0, nk, g, d0, lane, Mc, Lc, Ac);
    }
    if (has_gate) gate_factors(gw, a.gate_ref, gs);
    write_out(a.out, a.out_bf16, orow, d0, has_gate, gs, Lc, Ac);
    if (lane == 0) *ctr = 0;
}

// ---------------------------------------------------------------------------

int launch_quantize(const QuantizeArgs& a, void* stream) {
    const unsigned grid = (unsigned)a.n_blocks * a.p.n_layers * 2 * kKvHeads;
    hipLaunchKernelGGL(quantize_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int launch_gather_q8(const GatherQ8Args& a, void* stream) {
    hipLaunchKernelGGL(gather_q8_kernel, dim3((unsigned)a.n_items * 8), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int launch_decode_q8(const DecodeQ8Args& a, void* stream) {
    hipLaunchKernelGGL(decode_q8_kernel, dim3(a.per_xcd * 8), dim3(kWaves * 64), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

}  // namespace kvc
