// Acceptance of a drafted path: per stream, the rows of the accepted nodes move to the slots behind
// the cached ones, in every layer and head group, K and V; then the length grows.
//
// Bound by latency at a session's sizes and by memory for a batch (each moved row read and written
// once). A thread owns one 16-byte column of a (stream, block, K or V) and takes the path's rows in
// order, kBatch loads ahead of their stores: nodes rise, so node[j] >= j and no store comes before
// a load that needs its slot, and columns share no byte, so no thread waits for another. Measured (one
// B200): 512 paths in 9 layers, 14 us on the GPU, 1 to 2 of them a stream's CTAs counting one another.
#include "common.cuh"
#include "score.h"

namespace ptts {
namespace {

constexpr int kBatch = 8, kThreads = 128;

__device__ __forceinline__ void accept(const AcceptArgs& a, const int32_t* list) {
    const int i = blockIdx.x, sid = list[i], len = list[a.n + i];
    const int32_t* offsets = list + 2 * a.n;
    const int from = offsets[i], count = offsets[i + 1] - from;
    const int32_t* node = offsets + a.n + 1 + from;
    const bool first = blockIdx.y == 0 && threadIdx.x == 0;
    // The nodes lie behind the device's length: where that is not the host's, the path is refused.
    if (sid < 0 || sid >= a.streams || len < 0 || *const_cast<volatile int32_t*>(a.lengths + sid) != len) {
        if (first) set_error(a.err, DEV_ERR_BOUNDS);
        return;
    }
    if (count > 0 && len + node[count - 1] >= a.capacity) {
        if (first) set_error(a.err, DEV_ERR_CAPACITY);
        return;
    }
    // All of the stream's CTAs come here or none: the one that finds the others' reads done writes the length.
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        if (atomicAdd(a.arrived + sid, 1) == (int)gridDim.y - 1) {
            a.lengths[sid] = len + count;
            a.arrived[sid] = 0;
        }
    }
    const int c = blockIdx.y * blockDim.x + threadIdx.x;
    if (c >= 2 * a.blocks * a.row_vec) return;
    const int b = c / a.row_vec;
    uint4* base = static_cast<uint4*>(b < a.blocks ? a.k_cache : a.v_cache) + (b % a.blocks) * a.block_vec +
                  sid * a.stream_vec + (long long)len * a.row_vec + c % a.row_vec;
    for (int j0 = 0; j0 < count; j0 += kBatch) {
        uint4 x[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (j0 + j < count && node[j0 + j] != j0 + j) x[j] = base[(long long)node[j0 + j] * a.row_vec];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (j0 + j < count && node[j0 + j] != j0 + j) base[(long long)(j0 + j) * a.row_vec] = x[j];
    }
}

__global__ void __launch_bounds__(kThreads) accept_kernel(AcceptArgs a, const int32_t* __restrict__ list) {
    grid_dep_wait();
    grid_dep_launch();
    accept(a, list);
}

__global__ void __launch_bounds__(kThreads) accept_inline_kernel(AcceptArgs a, const __grid_constant__ AcceptInline l) {
    grid_dep_wait();
    grid_dep_launch();
    accept(a, l.list);
}

dim3 accept_grid(const AcceptArgs& a) { return dim3(a.n, (2 * a.blocks * a.row_vec + kThreads - 1) / kThreads); }

}  // namespace

void launch_accept(const AcceptArgs& a, const int32_t* list_dev, cudaStream_t s) {
    launch_k(accept_kernel, accept_grid(a), dim3(kThreads), 0, s, a, list_dev);
}

void launch_accept_inline(const AcceptArgs& a, const AcceptInline& list, cudaStream_t s) {
    launch_k(accept_inline_kernel, accept_grid(a), dim3(kThreads), 0, s, a, list);
}

}  // namespace ptts
