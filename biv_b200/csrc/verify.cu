// Drafted tokens against the target's probabilities: what is accepted, and one token from what is left.
//
// Bytes of one row of p (and of q) a request bound it, and for few requests the way to memory and back.  A request
// has a cluster of thread blocks, each with a part of the vocabulary.  Every block finds the first draft that fails by
// itself (a handful of values), sums its part's weights in f64 by segments of a warp's width, and learns the other
// blocks' sums through distributed shared memory; the block that the drawn weight falls into looks its segment
// up again (it is in the caches) and walks it in the vocabulary's order.  So the rows come from memory once and no
// block waits for one outside its cluster, which the hardware schedules together.
//
// 64 requests of 131072 bf16 values of p and q (33.5 MB): 10.5 us, some 2 of them the way to the drafts and their values, 5 the rows,
// 1 to 2 the sums' exchange and as much the search; one request 8.3 us, 250 of 32003 f32 values 11.2 (all from memory).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "rows_of.h"
#include "verify.cuh"

namespace bivmoe {

namespace {

namespace cg = cooperative_groups;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kSegment = 1024;                   // values whose sum is kept by itself: 32 to a lane
constexpr int kMostSegments = 5000;              // of a block

template <class T> __device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
    else return __bfloat162float(v);
}

// The weight of a token: what p has over q, or, without q, p but for the draft.
template <class T> struct Weights {
    const T *p, *q;                              // q null: p alone
    int vocab, without;                          // the token that has no weight, or -1
    bool together;                               // p and q lie alike within 16 bytes
    static constexpr int kPer = 16 / sizeof(T);

    __device__ __forceinline__ float at(int t) const {
        const float w = to_f32(p[t]) - (q ? to_f32(q[t]) : 0.0f);
        return t != without && w > 0.0f ? w : 0.0f;
    }
    // A piece of 16 bytes of a row; places outside the vocabulary are zeros.
    __device__ __forceinline__ uint4 piece(const T* row, int t) const {
        if (t >= 0 && t + kPer <= vocab) return *(const uint4*)(row + t);
        uint4 x = make_uint4(0, 0, 0, 0);
        if (t < vocab && t + kPer > 0) {             // a row's first or last
#pragma unroll
            for (int e = 0; e < kPer; e++)
                if (t + e >= 0 && t + e < vocab) ((T*)&x)[e] = row[t + e];
        }
        return x;
    }
    // A segment's values that a lane has, from `t` on and 32 lanes' pieces apart, or next to one another; p is aligned at t.
    template <int APART> __device__ __forceinline__ double sum(int t) const {
        constexpr int N = 32 / kPer;                 // pieces
        double s = 0.0;
        if (q && !together) {
#pragma unroll 1
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int e = 0; e < kPer; e++) {
                    const int u = t + i * APART + e;
                    if (u >= 0 && u < vocab) s += (double)at(u);
                }
            return s;
        }
        // (The row's ends apart, so that all loads of the others set out together: 250 rows of 32003 f32 took 17 us where the ends were
        // loaded value by value, and 64 of 131072 bf16 with q 14 and not 10.5 where every piece asked for its place.)
        uint4 a[N], b[N];
        if (t >= 0 && t + (N - 1) * APART + kPer <= vocab) {
#pragma unroll
            for (int i = 0; i < N; i++) a[i] = *(const uint4*)(p + t + i * APART);
            if (q)
#pragma unroll
                for (int i = 0; i < N; i++) b[i] = *(const uint4*)(q + t + i * APART);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) a[i] = piece(p, t + i * APART);
            if (q)
#pragma unroll
                for (int i = 0; i < N; i++) b[i] = piece(q, t + i * APART);
        }
        if (q) {
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int e = 0; e < kPer; e++) s += (double)fmaxf(to_f32(((const T*)&a[i])[e]) - to_f32(((const T*)&b[i])[e]), 0.0f);   // (NaN: zero)
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int e = 0; e < kPer; e++) s += t + i * APART + e != without ? (double)fmaxf(to_f32(((const T*)&a[i])[e]), 0.0f) : 0.0;
        }
        return s;
    }
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

template <class T> __global__ void __launch_bounds__(kThreads, 4) verify_kernel(const __grid_constant__ bivmoe_verify_args a) {
    extern __shared__ double segments[];
    __shared__ double room[kWarps], totals[2][16];
    pdl_enter();
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int blocks = cluster.num_blocks(), rank = cluster.block_rank(), b = blockIdx.x / blocks;
    // that all blocks of the cluster have begun is waited for before the first writes into another
    if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    const RowsOf rows = rows_of(a.first[b], a.first[b + 1], a.n_tokens);
    const int first = rows.first, n = rows.n;
    const T *p = (const T*)a.p, *q = (const T*)a.q;
    // every warp for itself: the first draft that fails
    int kept = max(n - 1, 0);
    for (int i0 = 0; i0 < n - 1; i0 += 32) {
        const int i = i0 + lane;
        bool good = true;
        if (i < n - 1) {
            const int64_t r = first + i;
            const int d = a.tokens[r + 1];
            const double u = a.uniform[r];
            good = d >= 0 && d < a.vocab;
            if (good) good = (q ? u * (double)to_f32(q[r * a.q_stride + d]) : u) < (double)to_f32(p[r * a.p_stride + d]);
        }
        const unsigned bad = __ballot_sync(0xffffffffu, !good);
        if (bad) {
            kept = i0 + __ffs(bad) - 1;
            break;
        }
    }
    if (rank == 0 && tid == 0) {
        a.accepted[b] = kept;
        if (a.kept) a.kept[b] = a.length[b] - max(n - 1 - kept, 0);
        if (!n) a.token[b] = -1;
    }
    if (blocks > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (!n) return;                              // the whole cluster
    const int64_t r = first + kept;
    bool rest = kept < n - 1;                    // what p has over q; else p
    Weights<T> w{p + r * a.p_stride, rest && q ? q + r * a.q_stride : nullptr, a.vocab, rest && !q ? a.tokens[r + 1] : -1, false};
    const int lead = (int)((uintptr_t)w.p % 16 / sizeof(T));
    w.together = w.q && (uintptr_t)w.q % 16 == (uintptr_t)w.p % 16;
    // segments of the row, from the boundary before its start on; a block's part of them
    const int all = (lead + a.vocab + kSegment - 1) / kSegment;
    const int s0 = (int)((int64_t)all * rank / blocks), s1 = (int)((int64_t)all * (rank + 1) / blocks);
    double sum = 0.0;
    const double* parts = totals[0];
    for (int turn = 0;; turn++) {
        for (int s = s0 + warp; s < s1; s += kWarps) {
            const double x = warp_sum(w.template sum<32 * Weights<T>::kPer>(s * kSegment - lead + lane * w.kPer));
            if (lane == 0) segments[s - s0] = x;
        }
        __syncthreads();
        double x = 0.0;
        for (int s = tid; s < s1 - s0; s += kThreads) x += segments[s];
        x = warp_sum(x);
        if (lane == 0) room[warp] = x;
        __syncthreads();
        parts = totals[turn];
        if (tid < blocks) {                      // this block's sum into every block of the cluster
            x = 0.0;
            for (int i = 0; i < kWarps; i++) x += room[i];
            *cluster.map_shared_rank(&totals[turn][rank], tid) = x;
        }
        if (blocks > 1) cluster.sync();
        else __syncthreads();
        sum = 0.0;
        for (int i = 0; i < blocks; i++) sum += parts[i];
        if (sum > 0.0 || !rest) break;
        rest = false;                            // no weight is left: p itself
        w.q = nullptr;
        w.without = -1;
    }
    if (!(sum > 0.0)) {
        if (rank == 0 && tid == 0) a.token[b] = -1;
        return;
    }
    // The block that the drawn weight falls into, or, where rounding leaves none, the last that holds any: all blocks
    // take the same sums in the same order, so that one of them finds itself.  So then for its segments, and a lane's 32
    // values of the segment, in the vocabulary's order.
    const double drawn = (double)a.sample[b] * sum;
    double upto = 0.0, before = 0.0;
    int owner = -1, last = 0;
    double last_before = 0.0;
    for (int i = 0; i < blocks && owner < 0; i++) {
        if (parts[i] > 0.0) { last = i; last_before = upto; }
        before = upto;
        upto += parts[i];
        if (upto > drawn) owner = i;
    }
    if (owner < 0) { owner = last; before = last_before; }
    if (rank != owner || warp) return;
    upto = before;
    int found = -1;
    last = 0;
    last_before = before;
    for (int s = 0; s < s1 - s0 && found < 0; s++) {
        if (segments[s] > 0.0) { last = s; last_before = upto; }
        before = upto;
        upto += segments[s];
        if (upto > drawn) found = s;
    }
    if (found < 0) { found = last; before = last_before; }
    const int t0 = (s0 + found) * kSegment - lead + lane * 32;
    auto weight = [&](int t) { return t >= 0 && t < a.vocab ? (double)w.at(t) : 0.0; };
    const double mine = w.template sum<Weights<T>::kPer>(t0);
    double end = mine;                           // sums up to a lane's end
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += x;
    }
    double start = __shfl_up_sync(0xffffffffu, end, 1);
    start = before + (lane ? start : 0.0);
    unsigned over = __ballot_sync(0xffffffffu, mine > 0.0 && before + end > drawn);
    const unsigned any = __ballot_sync(0xffffffffu, mine > 0.0);
    const int of = over ? __ffs(over) - 1 : 31 - __clz(any | 1);
    // its values, one to a lane
    const int t = __shfl_sync(0xffffffffu, t0, of) + lane;
    const double x = weight(t);
    end = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += y;
    }
    start = __shfl_sync(0xffffffffu, start, of);
    over = __ballot_sync(0xffffffffu, x > 0.0 && start + end > drawn);
    const unsigned some = __ballot_sync(0xffffffffu, x > 0.0);
    if (lane == (over ? __ffs(over) - 1 : 31 - __clz(some | 1))) a.token[b] = t;
}

template <class T> cudaError_t launch(const bivmoe_verify_args& a, int blocks, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.n_seq * blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = ((a.vocab + 2 * kSegment) / kSegment / blocks + 2) * sizeof(double);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_mode() != 0 ? 2 : 1;
    count_launch();
    return cudaLaunchKernelEx(&cfg, verify_kernel<T>, a);
}

}  // namespace

cudaError_t launch_verify(const bivmoe_verify_args& a, int sm_count, cudaStream_t stream) {
    // Blocks to a request: as many as run at once (four to an SM, less an eighth: a cluster's blocks share a part of the chip, and 148 clusters
    // of four took turns, 19.3 us for 131072 bf16 values each, by two 17.3), each with some segments; and as many as have room for
    // their segments' sums in shared memory.  (us with one, two, four, eight: one request of 100003 values 18.7, 13.8, 10.7, 9.7; 64 of 131072
    // 28, 18, 13, 10.5; 250 of 32003, of which four and more do not run at once, 18, 17, 25, 40; before its ends were loaded together.)
    int blocks = 1;
    while (blocks < 8 && (((int64_t)a.n_seq * blocks * 2 * 2 <= 7 * sm_count && a.vocab >= blocks * 2 * 2 * kSegment) ||
                          a.vocab / kSegment / blocks > kMostSegments))
        blocks *= 2;
    switch (a.ggml_type) {
        case BIVMOE_F32: return launch<float>(a, blocks, stream);
        case BIVMOE_F16: return launch<__half>(a, blocks, stream);
        default: return launch<__nv_bfloat16>(a, blocks, stream);
    }
}

}  // namespace bivmoe
