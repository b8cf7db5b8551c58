// kvc_fork_kernels.h -- copies of recurrent states and block-table rows for
// kvc_seq_fork and kvc_seq_reorder (included by kvc_kernels.hip).
#pragma once

namespace kvc {

// The first n_rows workgroups copy a block-table row each, the others pieces of
// the states: a piece is read once and stored to every sequence that gets it.
// Nothing is both read and written (a destination is nobody's source).  HBM-bound:
// 52.7 MB read a source and written a copy; one state to four sequences 48 us (5.4
// TB/s read + written), 13 copies of 5 163 us (5.8).  A thread moves one 16-B piece: 2,
// 4 and 8 took 168, 169 and 193 us for the 163.  Loads and stores are nontemporal: the
// states are larger than the caches, and the K/V in them stays (time the same without).
__global__ __launch_bounds__(256) void fork_kernel(ForkArgs a) {
    int b = blockIdx.x;
    if (b < a.n_rows) {
        const int32_t* src = a.table + (size_t)a.row_src[b] * a.table_stride;
        int32_t* dst = a.table + (size_t)a.row_dst[b] * a.table_stride;
        for (int i = threadIdx.x; i < a.row_len[b]; i += 256) dst[i] = src[i];
        return;
    }
    b -= a.n_rows;
    const int p = b / a.wgs_per_state;
    const size_t n = (size_t)a.state_bytes / 16;
    const size_t u = (size_t)(b - p * a.wgs_per_state) * 256 + threadIdx.x;
    if (u >= n) return;
    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.state + (size_t)a.src[p] * a.state_bytes) + u);
    for (int d = a.dst_begin[p]; d < a.dst_begin[p + 1]; d++)
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(a.state + (size_t)a.dst[d] * a.state_bytes) + u);
}

int launch_fork(const ForkArgs& a, void* stream) {
    ForkArgs f = a;
    f.wgs_per_state = (int32_t)((a.state_bytes / 16 + 255) / 256);
    const int64_t grid = a.n_rows + (int64_t)a.n_src * f.wgs_per_state;
    if (grid <= 0) return 0;
    if (grid > INT32_MAX) return (int)hipErrorInvalidConfiguration;
    hipLaunchKernelGGL(fork_kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, f);
    return (int)hipGetLastError();
}

}  // namespace kvc
