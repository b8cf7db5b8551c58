// kvc_beam_kernels.h -- beam search's choice: of each group (prompt) the n_out
// greatest of score_b + x_bt - log sum_u exp x_bu over its beams b and tokens t, in
// order (included by kvc_kernels.hip).
//
// Within a beam the order is that of the logits, so the first launch needs one pass
// over them: the maximum of every 256-token segment, and the sum of exponentials, in 32
// bits (added pairwise; the second launch adds the chunks' in 64, 0.2 us of it).
// The n_out greatest values of a group lie in the n_out segments with the greatest
// maxima (ties: the lower beam, then the lower segment): a value in any other
// segment has n_out segment maxima before it.  So the second launch, a workgroup per
// group, chooses among the maxima and reads few segments again.
//
// Measured: 32 groups of 8 beams of 151936 bf16 logits, 16 of each 23.3 us: the first
// launch 15.2 for 77.8 MB (5.1 TB/s; its VALU is busy for 10 of them, four tenths of
// that with the exponentials), the second 8.6, a chain of some ten trips to memory and
// barriers that a workgroup per group cannot hide.  One group of 4 beams 9.4: 2.8 + 6.7.
#pragma once

namespace kvc {

constexpr float kLog2e = 1.4426950408889634f;

// 16 B at any element's address: rows are cut by token, not by address, so that equal
// rows have equal sums wherever they lie.  The hardware takes such loads whole; of a
// wave's 1024 B they touch nine 128-B lines instead of eight.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <bool BF16>
__device__ __forceinline__ float beam_logit(const void* row, int t) {
    const float x = BF16 ? bf16f(static_cast<const uint16_t*>(row)[t]) : static_cast<const float*>(row)[t];
    return x != x ? -INFINITY : x;
}

__device__ __forceinline__ float beam_clean(float x) { return x != x ? -INFINITY : x; }

// A lane's 16 B of a row from token t on; -inf behind the row's end.
template <bool BF16>
__device__ __forceinline__ u32x4 beam_load(const uint8_t* row, int64_t t, int vocab) {
    constexpr int E = BF16 ? 8 : 4;
    if (t + E <= vocab) return *reinterpret_cast<const u32x4_any*>(row + t * (BF16 ? 2 : 4));
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (BF16) {
            const uint16_t* x = reinterpret_cast<const uint16_t*>(row);
            const uint32_t lo = t + 2 * i < vocab ? x[t + 2 * i] : 0xFF80u;
            const uint32_t hi = t + 2 * i + 1 < vocab ? x[t + 2 * i + 1] : 0xFF80u;
            w[i] = lo | hi << 16;
        } else {
            w[i] = t + i < vocab ? reinterpret_cast<const uint32_t*>(row)[t + i] : 0xFF800000u;
        }
    }
    return w;
}
template <bool BF16>
__device__ __forceinline__ float beam_word(const u32x4& w, int i) {
    if constexpr (BF16) return i & 1 ? bf16hi(w[i / 2]) : bf16lo(w[i / 2]);
    return __uint_as_float(w[i]);
}

// One chunk of a row: 4 waves x STEPS loads of 16 B a lane, all in flight at once.
// A segment's lanes are neighbours, and STEPS loads of theirs cover it.  A workgroup
// per chunk: loops over chunks with the next loads in flight took 16-21 us for the 15.2
// above.  STEPS 1, 2, 4, 8: 19.4, 15.5, 15.2, 16.2 us there, 2.8, 3.2, 4.1, 5.7 for one
// group of 4 beams.
template <bool BF16, int STEPS>
__global__ __launch_bounds__(256) void beam_max_kernel(BeamArgs a) {
    constexpr int E = BF16 ? 8 : 4;                    // tokens of a lane's load
    constexpr int kSegLanes = kBeamSeg / (E * STEPS);  // 8 to 64
    __shared__ float2 red[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = blockIdx.y;
    const uint8_t* base = static_cast<const uint8_t*>(a.logits) + row * (size_t)a.stride * (BF16 ? 2 : 4);
    const int64_t j = ((int64_t)blockIdx.x * 4 + wave) * (64 / kSegLanes) + lane / kSegLanes;  // the lane's segment
    const int64_t t0 = j * kBeamSeg + lane % kSegLanes * E;
    u32x4 w[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; k++) w[k] = beam_load<BF16>(base, t0 + k * kSegLanes * E, a.vocab);
    const auto logit = [&](int k, int i) __attribute__((always_inline)) { return beam_word<BF16>(w[k], i); };
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < STEPS; k++)
#pragma unroll
        for (int i = 0; i < E; i++) m = fmaxf(m, logit(k, i));
    float me = m == -INFINITY ? 0.f : m;
    // the lane's exponentials, added pairwise: log2 of their number roundings, not that
    // many, and small ones beside a 1 are not lost one by one
    const auto sum = [&](auto&& x) __attribute__((always_inline)) {
        float e[STEPS * E];
#pragma unroll
        for (int k = 0; k < STEPS * E; k++) e[k] = fast_exp2((x(k / E, k % E) - me) * kLog2e);
#pragma unroll
        for (int n = 1; n < STEPS * E; n *= 2)
#pragma unroll
            for (int k = 0; k < STEPS * E; k += 2 * n) e[k] += e[k + n];
        return e[0];
    };
    float s = sum(logit);
    if (s != s) {  // a NaN counts as -inf; so does +inf here, whose sum nobody reads
        const auto clean = [&](int k, int i) __attribute__((always_inline)) { return beam_clean(logit(k, i)); };
        m = -INFINITY;
#pragma unroll
        for (int k = 0; k < STEPS; k++)
#pragma unroll
            for (int i = 0; i < E; i++) m = fmaxf(m, clean(k, i));
        me = m == -INFINITY ? 0.f : m;
        s = sum(clean);
    }
    float seg = m;  // over the segment's lanes
    seg = fmaxf(seg, dpp<kDppXor1>(seg));
    seg = fmaxf(seg, dpp<kDppXor2>(seg));
    seg = fmaxf(seg, dpp<kDppHalfMirror>(seg));
    if constexpr (kSegLanes >= 16) seg = fmaxf(seg, dpp<kDppRowRor8>(seg));
    if constexpr (kSegLanes >= 32) seg = max_xor16(seg);
    if constexpr (kSegLanes == 64) seg = max_xor32(seg);
    if (lane % kSegLanes == 0 && j < a.n_seg) a.seg_max[row * a.n_seg + j] = seg;
    const float wm = wave_max(m), we = wm == -INFINITY ? 0.f : wm;
    s = wave_sum(s * fast_exp2((m - we) * kLog2e));
    if (lane == 0) red[wave] = make_float2(wm, s);
    __syncthreads();
    if (threadIdx.x == 0) {
        const float M = fmaxf(fmaxf(red[0].x, red[1].x), fmaxf(red[2].x, red[3].x)), e = M == -INFINITY ? 0.f : M;
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] = red[i].y * fast_exp2((red[i].x - e) * kLog2e);
        *reinterpret_cast<float2*>(a.chunk_sum + (row * a.n_chunks + blockIdx.x) * 2) = make_float2(M, (t[0] + t[1]) + (t[2] + t[3]));
    }
}

template <int CTRL>
__device__ __forceinline__ double dpp64(double x) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, 0xF, 0xF, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ double wave_sum64(double x) {
    x += dpp64<kDppXor1>(x);
    x += dpp64<kDppXor2>(x);
    x += dpp64<kDppHalfMirror>(x);
    x += dpp64<kDppRowRor8>(x);
    uint32_t l = __double2loint(x), h = __double2hiint(x);
    auto lo = __builtin_amdgcn_permlane16_swap(l, l, false, false), hi = __builtin_amdgcn_permlane16_swap(h, h, false, false);
    x = __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
    l = __double2loint(x), h = __double2hiint(x);
    lo = __builtin_amdgcn_permlane32_swap(l, l, false, false), hi = __builtin_amdgcn_permlane32_swap(h, h, false, false);
    return __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
}

// e^(x - m), x <= m, as the hardware's exponential of the rounded argument and the
// first order of what rounding took from it: off by that exponential's 2^-23.  0
// for -inf (whose argument would leave NaN in the second part).
__device__ __forceinline__ double beam_scale(float x, float m) {
    const double y = fmax((double)x - (double)m, -300.0) * 1.4426950408889634;
    const float p = (float)y, e = fast_exp2(p);
    return (double)e + (double)(e * (float)(y - (double)p)) * 0.6931471805599453;
}

// log x of a finite x >= 1: the exponent's part and what rounding took from the
// mantissa in 64 bits, the rounded mantissa's by the hardware, off by 2^-24 at most.
__device__ __forceinline__ double beam_log(double x) {
    const int hi = __double2hiint(x);
    const double f = __hiloint2double((hi & 0xFFFFF) | 0x3FF00000, __double2loint(x));  // in [1, 2)
    const float c = (float)f, d = (float)(f - (double)c);
    return ((double)((hi >> 20) - 1023) + (double)__builtin_amdgcn_logf(c)) * 0.6931471805599453 +
           (double)(d * __builtin_amdgcn_rcpf(c));
}

// Doubles as integers of the same order; 0 for -inf, which is never chosen.
__device__ __forceinline__ uint64_t beam_key(double v) {
    if (!(v > -INFINITY)) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);  // (-0 is 0)
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double beam_value(uint64_t k) {
    return __longlong_as_double((int64_t)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

constexpr int kBeamThreads = 1024, kBeamWaves = kBeamThreads / 64;
constexpr int kBeamHeld = 8;      // a thread's segment maxima in registers
constexpr int kBeamCands = 1024;  // segments, then values, that are looked at one by one
struct BeamSmem {
    uint64_t cand[kBeamCands];   // key of a value, and where it is: beam << 32 | token
    uint64_t where[kBeamCands];
    double off[kBeamMaxBeams];   // score - log sum exp(x - max); -inf for a beam that gives nothing
    double max[kBeamMaxBeams];
    uint64_t red[2 * kBeamWaves];
    int32_t list[kBeamCands];    // chosen segments
    int32_t hist[kBeamThreads];
    int32_t wsum[kBeamWaves];
    float wmax[kBeamWaves];
    int32_t count, listed, kept, bin, above;
};

__device__ __forceinline__ int beam_scan(BeamSmem& sm, int x, int tid) {  // sum over threads >= tid
    const int lane = tid & 63, wave = tid >> 6;
    int v = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_down(v, d);
        v += lane + d < 64 ? y : 0;
    }
    if (lane == 0) sm.wsum[wave] = v;
    __syncthreads();
    for (int w = wave + 1; w < kBeamWaves; w++) v += sm.wsum[w];
    __syncthreads();
    return v;
}

template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int dpp_or_0(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
// Sum over the wave's lanes up to this one: by shifts within rows of 16, then of a
// row's last lane to the next row, and of lane 31 to the upper half.
__device__ __forceinline__ int wave_prefix(int x) {
    x += dpp_or_0<0x111>(x);
    x += dpp_or_0<0x112>(x);
    x += dpp_or_0<0x114>(x);
    x += dpp_or_0<0x118>(x);
    x += dpp_or_0<0x142, 0xA>(x);
    x += dpp_or_0<0x143, 0xC>(x);
    return x;
}

// Of n keys (0: none) the `want` greatest: those above *cut, and of those equal to
// it the first *ties.  All threads; want >= 1.
template <typename Key>
__device__ __forceinline__ void beam_cut(BeamSmem& sm, int n, int want, Key&& key, uint64_t* cut, int* ties) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t lo = ~0ull, hi = 0;
    int alive = 0;
    for (int p = tid; p < n; p += kBeamThreads) {
        const uint64_t k = key(p);
        if (k == 0) continue;
        alive++;
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
    }
#pragma unroll
    for (int d = 32; d; d /= 2) {
        const uint64_t l2 = __shfl_xor(lo, d), h2 = __shfl_xor(hi, d);
        lo = l2 < lo ? l2 : lo;
        hi = h2 > hi ? h2 : hi;
    }
    if (lane == 0) {
        sm.red[2 * wave] = lo;
        sm.red[2 * wave + 1] = hi;
    }
    const int total = beam_scan(sm, alive, tid);  // (thread 0's is the sum of all; its barriers order red)
    if (tid == 0) sm.above = total;
    for (int w = 0; w < kBeamWaves; w++) {
        lo = sm.red[2 * w] < lo ? sm.red[2 * w] : lo;
        hi = sm.red[2 * w + 1] > hi ? sm.red[2 * w + 1] : hi;
    }
    __syncthreads();
    if (sm.above <= want) {  // all that there are
        *cut = 1;
        *ties = n;
        __syncthreads();
        return;
    }
    // narrow [lo, hi] to the 1024th part that holds the want-th greatest, until it
    // is taken whole or is one value (4 rounds at least of 64 bits; 2 or 3 in use)
    int need = want;
    for (;;) {
        const uint64_t width = hi - lo;
        const int bits = width ? 64 - __clzll((long long)width) : 0;
        const int sh = bits > 10 ? bits - 10 : 0;
        __syncthreads();
        sm.hist[tid] = 0;
        __syncthreads();
        for (int p = tid; p < n; p += kBeamThreads) {
            const uint64_t k = key(p);
            if (k >= lo && k <= hi) atomicAdd(&sm.hist[(int)((k - lo) >> sh)], 1);
        }
        __syncthreads();
        const int h = sm.hist[tid];
        const int from = beam_scan(sm, h, tid);  // in this part and above
        if (from >= need && from - h < need) {
            sm.bin = tid;
            sm.above = from - h;
            sm.count = h;
        }
        __syncthreads();
        const int bin = sm.bin, inside = sm.count;
        need -= sm.above;
        lo += (uint64_t)bin << sh;
        const uint64_t top = lo + ((1ull << sh) - 1);
        hi = top < hi ? top : hi;
        if (inside == need || sh == 0) break;
    }
    __syncthreads();
    // one value left: its first `need` places; a part taken whole: all from lo on
    if (lo == hi) {
        *cut = lo;
        *ties = need;
    } else {
        *cut = lo;
        *ties = n;
    }
}

// emit(p) for the chosen of n keys, in no order.
template <typename Key, typename Emit>
__device__ __forceinline__ void beam_collect(BeamSmem& sm, int n, uint64_t cut, int ties, Key&& key, Emit&& emit) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (ties >= n) {
        for (int p = tid; p < n; p += kBeamThreads) {
            const uint64_t k = key(p);
            if (k >= cut && k) emit(p, k);
        }
        return;
    }
    int before = 0;  // equal ones in earlier rounds
    for (int p0 = 0; p0 < n; p0 += kBeamThreads) {
        const int p = p0 + tid;
        const uint64_t k = p < n ? key(p) : 0;
        const bool eq = k == cut;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(eq);
        if (lane == 0) sm.wsum[wave] = __popcll(mask);
        __syncthreads();
        int r = before + __popcll(mask & ((1ull << lane) - 1));
        for (int w = 0; w < kBeamWaves; w++) {
            if (w < wave) r += sm.wsum[w];
            before += sm.wsum[w];
        }
        if (k > cut || (eq && r < ties)) emit(p, k);
        __syncthreads();
    }
}

// Distances from the greatest value, 32 parts to an octave from 2^-16 to 2^16.
__device__ __forceinline__ int beam_part(double top, double v) {
    const float d = (float)(top - v);
    const int i = (int)(__float_as_uint(d > 0.f ? d : 0.f) >> 18) - (111 << 5);
    return i < 0 ? 0 : i > 1023 ? 1023 : i;
}

// A workgroup per group.  A histogram of the threads' greatest segment maxima, by their
// distance from the greatest of all, finds a part that n_out of them reach; the values that reach it are among
// those segments' and are few, since a part is 3 % of a distance: they are ranked by
// counting.  Where they are more than can be held (rows of one level, say), the
// n_out greatest maxima and then values are found exactly, equal ones by place.
template <bool BF16>
__global__ __launch_bounds__(kBeamThreads) void beam_select_kernel(BeamArgs a) {
    __shared__ BeamSmem sm;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t row0 = (size_t)blockIdx.x * a.n_beams;
    const int n_seg = a.n_seg, n = a.n_beams * n_seg;
    const float* seg = a.seg_max + row0 * n_seg;
    float held[kBeamHeld];
#pragma unroll
    for (int i = 0; i < kBeamHeld; i++) {
        const int p = i * kBeamThreads + tid;
        held[i] = p < n ? seg[p] : -INFINITY;
    }
    sm.hist[tid] = 0;
    if (tid == 0) {
        sm.count = sm.listed = sm.kept = 0;
        sm.bin = kBeamThreads - 1;
    }
    // A value is (score - log sum exp(x - max)) + (x - max), in 64 bits: large logits
    // cancel before the small sums join them.
    for (int b = wave; b < a.n_beams; b += kBeamWaves) {
        const float2* cs = reinterpret_cast<const float2*>(a.chunk_sum) + (row0 + b) * (size_t)a.n_chunks;
        const float score = a.scores ? a.scores[row0 + b] : 0.f;
        const float2 none = make_float2(-INFINITY, 0.f);
        const float2 c0 = lane < a.n_chunks ? cs[lane] : none, c1 = lane + 64 < a.n_chunks ? cs[lane + 64] : none;
        float m = fmaxf(c0.x, c1.x);
        for (int c = lane + 128; c < a.n_chunks; c += 64) m = fmaxf(m, cs[c].x);
        m = wave_max(m);
        const bool fine = m > -INFINITY && m < INFINITY;
        double s = 0.0;
        if (fine) {
            s = (double)c0.y * beam_scale(c0.x, m) + (double)c1.y * beam_scale(c1.x, m);
            for (int c = lane + 128; c < a.n_chunks; c += 64) s += (double)cs[c].y * beam_scale(cs[c].x, m);
        }
        s = wave_sum64(s);
        if (lane == 0) {
            sm.off[b] = fine && score > -INFINITY && score < INFINITY ? score - beam_log(s) : -INFINITY;
            sm.max[b] = fine ? m : 0.0;
        }
    }
    __syncthreads();
    const float per_seg = 1.f / (float)n_seg;
    // (the quotient is at least 0.5 / n_seg from an integer, and off by 2^-22 of itself)
    const auto beam_of = [&](int p) {
        return p < 1 << 20 ? (int)(((float)p + 0.5f) * per_seg) : (int)((unsigned)p / (unsigned)n_seg);
    };
    const auto value_of = [&](int b, float x) { return sm.off[b] + ((double)x - sm.max[b]); };
    double val[kBeamHeld];
    double mine = -INFINITY;  // the thread's greatest
#pragma unroll
    for (int i = 0; i < kBeamHeld; i++) {
        const int p = i * kBeamThreads + tid;
        val[i] = -INFINITY;
        if (i * kBeamThreads < n) val[i] = value_of(p < n ? beam_of(p) : 0, held[i]);
        mine = val[i] > mine ? val[i] : mine;
    }
    for (int p = kBeamHeld * kBeamThreads + tid; p < n; p += kBeamThreads) {
        const double v = value_of(beam_of(p), seg[p]);
        mine = v > mine ? v : mine;
    }
    float top = wave_max(fmaxf((float)mine, -__FLT_MAX__));
    if (lane == 0) sm.wmax[wave] = top;
    __syncthreads();
    top = wave_max(sm.wmax[lane % kBeamWaves]);
    if (mine > -INFINITY) atomicAdd(&sm.hist[beam_part(top, mine)], 1);
    __syncthreads();
    const auto reached = [&] {  // the first part that n_out of those counted reach, or the last
        const int h = sm.hist[tid];
        int to = wave_prefix(h);  // in this part and before it
        if (lane == 63) sm.wsum[wave] = to;
        __syncthreads();
        for (int w = 0; w < wave; w++) to += sm.wsum[w];
        if (to >= a.n_out && to - h < a.n_out) sm.bin = tid;
        __syncthreads();
        return sm.bin;
    };
    const int last = reached();
    const auto choose = [&](int p, double v) {
        if (!(v > -INFINITY) || beam_part(top, v) > last) return;
        const int c = atomicAdd(&sm.listed, 1);
        if (c < kBeamCands) sm.list[c] = p;
    };
    if (mine > -INFINITY && beam_part(top, mine) <= last) {
#pragma unroll
        for (int i = 0; i < kBeamHeld; i++) choose(i * kBeamThreads + tid, val[i]);
        for (int p = kBeamHeld * kBeamThreads + tid; p < n; p += kBeamThreads) choose(p, value_of(beam_of(p), seg[p]));
    }
    __syncthreads();
    const size_t esz = BF16 ? 2 : 4;
    const uint8_t* rows = static_cast<const uint8_t*>(a.logits) + row0 * (size_t)a.stride * esz;
    const auto place = [&](int p, int i, int* b, int64_t* t) -> const uint8_t* {
        *b = beam_of(p);
        *t = (int64_t)(p - *b * n_seg) * kBeamSeg + i;
        return rows + (size_t)*b * (size_t)a.stride * esz;
    };
    int n_list = sm.listed, n_cand = kBeamCands + 1;
    if (n_list <= kBeamCands) {
        constexpr int E = BF16 ? 8 : 4, kLanes = kBeamSeg / E;
        const auto walk = [&](int to, auto&& f) {  // f(beam, token, value, part) of the values that reach part `to`
            for (int k = tid / kLanes; k < n_list; k += kBeamThreads / kLanes) {
                int b;
                int64_t t;
                const uint8_t* row = place(sm.list[k], tid % kLanes * E, &b, &t);
                const u32x4 w = beam_load<BF16>(row, t, a.vocab);
#pragma unroll
                for (int i = 0; i < E; i++) {
                    const double v = value_of(b, beam_clean(beam_word<BF16>(w, i)));
                    const int part = beam_part(top, v);
                    if (v > -INFINITY && part <= to) f(b, (int)(t + i), v, part);
                }
            }
        };
        const auto keep = [&](int32_t& count, uint64_t key, uint64_t where) {
            const int c = atomicAdd(&count, 1);
            if (c < kBeamCands) {
                sm.cand[c] = key;
                sm.where[c] = where;
            }
        };
        const auto place_of = [](int b, int t) { return (uint64_t)b << 32 | (uint32_t)t; };
        walk(last, [&](int b, int t, double v, int) { keep(sm.count, beam_key(v), place_of(b, t)); });
        __syncthreads();
        n_cand = sm.count;
        if (n_cand > 2 * a.n_out + 64) {
            // few segments, or many values in each that reach the part: count again,
            // among the values (ranking costs the square: 1024 of them 30 us)
            const bool here = n_cand <= kBeamCands;
            const uint64_t key = here && tid < n_cand ? sm.cand[tid] : 0, where = here && tid < n_cand ? sm.where[tid] : 0;
            const int part = key ? beam_part(top, beam_value(key)) : kBeamThreads;
            __syncthreads();
            sm.hist[tid] = 0;
            if (tid == 0) sm.bin = kBeamThreads - 1;
            __syncthreads();
            if (here) {
                if (key) atomicAdd(&sm.hist[part], 1);
            } else {
                walk(last, [&](int, int, double, int p) { atomicAdd(&sm.hist[p], 1); });
            }
            __syncthreads();
            const int to = reached();
            if (!here)
                walk(to, [&](int b, int t, double v, int) { keep(sm.kept, beam_key(v), place_of(b, t)); });
            else if (part <= to)
                keep(sm.kept, key, where);
            __syncthreads();
            n_cand = sm.kept;
        }
    }
    if (n_cand > kBeamCands) {
        const auto seg_key = [&](int p) { return beam_key(value_of(beam_of(p), seg[p])); };
        uint64_t cut;
        int ties;
        __syncthreads();
        beam_cut(sm, n, a.n_out, seg_key, &cut, &ties);
        if (tid == 0) sm.count = 0;
        __syncthreads();
        beam_collect(sm, n, cut, ties, seg_key, [&](int p, uint64_t) { sm.list[atomicAdd(&sm.count, 1)] = p; });
        __syncthreads();
        n_list = sm.count;
        if (tid < n_list) {  // in order of place
            const int p = sm.list[tid];
            int r = 0;
            for (int k = 0; k < n_list; k++) r += sm.list[k] < p;
            sm.hist[r] = p;
        }
        __syncthreads();
        if (tid < n_list) sm.list[tid] = sm.hist[tid];
        __syncthreads();
        const auto key = [&](int q) -> uint64_t {
            int b;
            int64_t t;
            const void* row = place(sm.list[q / kBeamSeg], q % kBeamSeg, &b, &t);
            return t >= a.vocab ? 0 : beam_key(value_of(b, beam_logit<BF16>(row, (int)t)));
        };
        beam_cut(sm, n_list * kBeamSeg, a.n_out, key, &cut, &ties);
        if (tid == 0) sm.count = 0;
        __syncthreads();
        beam_collect(sm, n_list * kBeamSeg, cut, ties, key, [&](int q, uint64_t v) {
            const int c = atomicAdd(&sm.count, 1);
            int b;
            int64_t t;
            place(sm.list[q / kBeamSeg], q % kBeamSeg, &b, &t);
            sm.cand[c] = v;
            sm.where[c] = (uint64_t)b << 32 | (uint32_t)t;
        });
        __syncthreads();
        n_cand = sm.count;
    }
    // in order: greatest first, then the lower beam, then the lower token; a value's
    // rank is counted by as many neighbouring lanes as there are threads for
    const size_t o = (size_t)blockIdx.x * a.n_out;
    const int lanes = n_cand <= 64 ? 16 : n_cand <= 256 ? 4 : 1, part = tid & (lanes - 1);
    const int c = n_cand <= 64 ? tid >> 4 : n_cand <= 256 ? tid >> 2 : tid;
    if (tid - lane < n_cand * lanes) {  // (the wave has some)
        const uint64_t v = c < n_cand ? sm.cand[c] : 0, w = c < n_cand ? sm.where[c] : 0;
        int r = 0;
        for (int k = part; k < n_cand; k += lanes) r += sm.cand[k] > v || (sm.cand[k] == v && sm.where[k] < w);
        if (lanes > 1) {
            r += dpp_or_0<kDppXor1>(r);
            r += dpp_or_0<kDppXor2>(r);
        }
        if (lanes > 4) {
            r += dpp_or_0<kDppHalfMirror>(r);
            r += dpp_or_0<kDppRowRor8>(r);
        }
        if (c < n_cand && part == 0 && r < a.n_out) {
            a.out_scores[o + r] = (float)beam_value(v);
            a.out_beams[o + r] = (int32_t)(w >> 32);
            a.out_tokens[o + r] = (int32_t)(uint32_t)w;
        }
    }
    if (tid >= n_cand && tid < a.n_out) {  // fewer than n_out
        a.out_scores[o + tid] = -INFINITY;
        a.out_beams[o + tid] = a.out_tokens[o + tid] = -1;
    }
}

int launch_beam_select(const BeamArgs& a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid(a.n_chunks, a.n_groups * a.n_beams);
    if (a.bf16 && a.steps == 4)
        hipLaunchKernelGGL((beam_max_kernel<true, 4>), grid, dim3(256), 0, st, a);
    else if (a.bf16)
        hipLaunchKernelGGL((beam_max_kernel<true, 1>), grid, dim3(256), 0, st, a);
    else if (a.steps == 4)
        hipLaunchKernelGGL((beam_max_kernel<false, 4>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((beam_max_kernel<false, 1>), grid, dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    if (a.bf16)
        hipLaunchKernelGGL(beam_select_kernel<true>, dim3(a.n_groups), dim3(kBeamThreads), 0, st, a);
    else
        hipLaunchKernelGGL(beam_select_kernel<false>, dim3(a.n_groups), dim3(kBeamThreads), 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace kvc
