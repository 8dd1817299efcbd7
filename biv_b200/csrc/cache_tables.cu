// Pages, slots and positions of new tokens, and the rotary store into the pages.
#include "cache.cuh"
#include "common.cuh"
#include "launch.cuh"

namespace bivmoe {

// ---- extend --------------------------------------------------------------------------------------
// Three exclusive sums over the requests (new tokens, new pages) decide everything else, and the
// requests are 1024 at most: every block makes the sums by itself (8 bytes a request from L2) and then
// fills its own part of the rows and of the new table entries, so that the call is one launch.
// A page that a row needs and that is new is read from the free list, not from the table, which
// another block may not have written yet.
// Bound by latency: launch, one load, the sums, one search, one load.
constexpr int kExtendThreads = 256;
constexpr int kExtendEach = kCacheSeqs / kExtendThreads;

struct ExtendCall {
    bivmoe_extend_args a;
    FastDiv page;
};

__device__ __forceinline__ int last_at_or_before(const int* first, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= v) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kExtendThreads) extend_kernel(ExtendCall c) {
    __shared__ int s_first[kCacheSeqs + 1], s_page[kCacheSeqs + 1], s_past[kCacheSeqs], s_have[kCacheSeqs];
    __shared__ int s_sum[2 * kExtendThreads / 32];
    const bivmoe_extend_args& a = c.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n_seq;
    const int count = max(min(*a.free_count, a.n_free), 0);
    int tokens = 0, pages = 0, add[kExtendEach], need[kExtendEach];
#pragma unroll
    for (int i = 0; i < kExtendEach; i++) {
        // consecutive requests to a thread: the sums over threads are then sums in the requests' order
        const int b = tid * kExtendEach + i;
        add[i] = need[i] = 0;
        if (b < n) {
            const int past = max(min(a.past[b], kCachePositions), 0);
            add[i] = max(min(a.added[b], kCacheTokens), 0);
            const int holds = (int)c.page.div(past + c.page.d - 1);
            const int have = a.held ? max(min(a.held[b], a.table_width), 0) : holds;
            need[i] = max((int)c.page.div(past + add[i] + c.page.d - 1) - have, 0);
            s_past[b] = past;
            s_have[b] = have;
            tokens += add[i];
            pages += need[i];
            if (blockIdx.x == 0) {
                a.length[b] = past + add[i];
                if (a.held_out) a.held_out[b] = have + need[i];
            }
        }
    }
    int xt = tokens, xp = pages;
    for (int d = 1; d < 32; d <<= 1) {
        const int yt = __shfl_up_sync(0xffffffffu, xt, d), yp = __shfl_up_sync(0xffffffffu, xp, d);
        if (lane >= d) { xt += yt; xp += yp; }
    }
    if (lane == 31) { s_sum[2 * warp] = xt; s_sum[2 * warp + 1] = xp; }
    __syncthreads();
    int bt = xt - tokens, bp = xp - pages, all_t = 0, all_p = 0;
    for (int i = 0; i < kExtendThreads / 32; i++) {
        if (i < warp) { bt += s_sum[2 * i]; bp += s_sum[2 * i + 1]; }
        all_t += s_sum[2 * i];
        all_p += s_sum[2 * i + 1];
    }
#pragma unroll
    for (int i = 0; i < kExtendEach; i++) {
        const int b = tid * kExtendEach + i;
        if (b < n) {
            s_first[b] = bt;
            s_page[b] = bp;
            if (blockIdx.x == 0) a.first[b] = bt;
        }
        bt += add[i];
        bp += need[i];
    }
    if (tid == 0) {
        s_first[n] = all_t;
        s_page[n] = all_p;
        if (blockIdx.x == 0) {
            a.first[n] = all_t;
            a.left[0] = max(count - all_p, 0);
            a.left[1] = max(all_p - count, 0);
        }
    }
    __syncthreads();
    const int step = gridDim.x * kExtendThreads, me = blockIdx.x * kExtendThreads + tid;
    for (int i = me; i < all_p; i += step) {
        const int b = last_at_or_before(s_page, n, i), at = s_have[b] + i - s_page[b];
        if (at < a.table_width) a.table[b * a.table_stride + at] = i < count ? a.free_pages[count - 1 - i] : -1;
    }
    for (int t = me; t < a.n_tokens; t += step) {
        int64_t slot = -1;
        int p = 0;
        if (t < all_t) {
            const int b = last_at_or_before(s_first, n, t);
            p = s_past[b] + t - s_first[b];
            const int at = (int)c.page.div(p);
            if (at < a.table_width) {
                const int i = s_page[b] + at - s_have[b];   // of the new pages
                const int page = at < s_have[b] ? a.table[b * a.table_stride + at] : i < count ? a.free_pages[count - 1 - i] : -1;
                if (page >= 0) slot = (int64_t)page * c.page.d + (p - at * (int)c.page.d);
            }
        }
        a.slots[t] = slot;
        a.positions[t] = p;
    }
}

cudaError_t launch_extend(const bivmoe_extend_args& a, int page_size, int sm_count, cudaStream_t stream) {
    ExtendCall c{a, FastDiv((uint32_t)page_size)};
    // a few rows a thread: more blocks only repeat the sums
    const int blocks = (int)min((int64_t)sm_count, ((int64_t)a.n_tokens + 2 * kExtendThreads - 1) / (2 * kExtendThreads) + 1);
    extend_kernel<<<blocks, kExtendThreads, 0, stream>>>(c);
    count_launch();
    return cudaGetLastError();
}

// ---- store ---------------------------------------------------------------------------------------
// (x, y) -> (x cos t - y sin t, x sin t + y cos t) for the pairs of the head's first n_rot values, t the
// token's position on the pair's axis times base^(-2i / n_rot).  A position times a frequency loses
// whole radians in f32 long before a cache is full (2^18 tokens: 0.01 rad), so the angle is made in
// f64, in turns, its whole turns taken off, and only the rest goes to f32 for the sine and cosine:
// once for each token and pair, shared by all heads.
// Bound by memory: a row is read once and written once, in 16-byte pieces.  A block takes a token at a
// time; the rows it needs are asked for before the angles are made.
constexpr int kStoreThreads = 256;
constexpr int kStoreDepth = 2;       // units a thread holds: one trip to memory for 512 units of 16 values

struct StoreCall {
    bivmoe_store_args a;
    RopePlan rope;
    FastDiv page;
    int heads, heads_kv, dim;
    bool wide;                       // 16-byte loads of q, k and v
};

template <class In> __device__ __forceinline__ void load8(const In* p, bool wide, float (&v)[8]) {
    if (wide) {
        constexpr int N = sizeof(In) / 2;            // 16-byte pieces
        uint4 w[N];
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = ((const uint4*)p)[i];
        const In* e = (const In*)w;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32(p[i]);
    }
}
template <class T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    uint4 w;
    w.x = pack2<T>(v[0], v[1]);
    w.y = pack2<T>(v[2], v[3]);
    w.z = pack2<T>(v[4], v[5]);
    w.w = pack2<T>(v[6], v[7]);
    *(uint4*)p = w;
}

// A unit is 16 values of a row of a head: two pieces of 8, `gap` values apart, that hold eight pairs
// (or, past n_rot and in v, nothing to turn).
template <class In, class T> struct Unit {
    const In* src;
    T* dst;
    int gap, pair;                   // pair: the first of the eight, or -1
    float x[8], y[8];
};

template <class In, class T, bool ADJACENT>
__global__ void __launch_bounds__(kStoreThreads) store_kernel(StoreCall c) {
    __shared__ float2 turn[kRopePairs];
    const bivmoe_store_args& a = c.a;
    const int tid = threadIdx.x, per_row = c.dim / 16, units = (c.heads + 2 * c.heads_kv) * per_row;
    const int pairs = c.rope.n_rot / 2, turned = c.rope.n_rot / 16;
    for (int t = blockIdx.x; t < a.n_tokens; t += gridDim.x) {
        const int64_t slot = a.slots[t];
        // a slot past 2^31 is past any pool that fits the device
        const int64_t page = slot >= 0 && slot >> 31 == 0 ? (int64_t)c.page.div((uint32_t)slot) : -1;
        const int at = (int)(slot - page * c.page.d);
        const bool kept = page >= 0 && page < a.k_pool.n_pages && page < a.v_pool.n_pages;
        for (int u0 = tid; u0 - tid < units; u0 += kStoreDepth * kStoreThreads) {
            Unit<In, T> unit[kStoreDepth];
#pragma unroll
            for (int i = 0; i < kStoreDepth; i++) {
                Unit<In, T>& u = unit[i];
                const int at_u = u0 + i * kStoreThreads, row = at_u / per_row, w = at_u - row * per_row;
                u.dst = nullptr;
                if (at_u >= units) continue;
                const bool is_q = row < c.heads, is_k = !is_q && row < c.heads + c.heads_kv;
                const int h = is_q ? row : is_k ? row - c.heads : row - c.heads - c.heads_kv;
                const bivmoe_rows& r = is_q ? a.q : is_k ? a.k : a.v;
                if (!is_q && !kept) continue;
                const bool turns = (is_q || is_k) && w < turned;
                const int off = !turns ? 16 * w : ADJACENT ? 16 * w : 8 * w;
                u.gap = turns && !ADJACENT ? pairs : 8;
                u.pair = turns ? 8 * w : -1;
                u.src = (const In*)r.data + t * r.stride_token + h * r.stride_head + off;
                const bivmoe_pool& p = is_k ? a.k_pool : a.v_pool;
                u.dst = is_q ? (T*)a.q_out.data + t * a.q_out.stride_token + h * a.q_out.stride_head + off
                             : (T*)p.data + page * p.stride_page + at * p.stride_token + h * p.stride_head + off;
                load8(u.src, c.wide, u.x);
                load8(u.src + u.gap, c.wide, u.y);
            }
            if (u0 == tid && pairs) {
                __syncthreads();             // the token before is done with its angles
                for (int i = tid; i < pairs; i += kStoreThreads) {
                    const double turns = (double)a.positions[c.rope.axis[i] * a.positions_stride + t] * c.rope.turns[i];
                    float s, co;
                    sincospif((float)(2.0 * (turns - rint(turns))), &s, &co);
                    turn[i] = make_float2(co, s);
                }
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < kStoreDepth; i++) {
                Unit<In, T>& u = unit[i];
                if (!u.dst) continue;
                if (u.pair >= 0) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float2 r = turn[u.pair + e];
                        float& x = ADJACENT ? (e < 4 ? u.x[2 * e] : u.y[2 * e - 8]) : u.x[e];
                        float& y = ADJACENT ? (e < 4 ? u.x[2 * e + 1] : u.y[2 * e - 7]) : u.y[e];
                        const float p = x * r.x - y * r.y, q = x * r.y + y * r.x;
                        x = p;
                        y = q;
                    }
                }
                store8(u.dst, u.x);
                store8(u.dst + u.gap, u.y);
            }
        }
    }
}

template <class In, class T> static void store_as(const StoreCall& c, int blocks, cudaStream_t stream) {
    if (c.rope.adjacent) store_kernel<In, T, true><<<blocks, kStoreThreads, 0, stream>>>(c);
    else store_kernel<In, T, false><<<blocks, kStoreThreads, 0, stream>>>(c);
}
template <class T> static void store_from(const StoreCall& c, int blocks, cudaStream_t stream) {
    switch (c.a.q.ggml_type) {
        case BIVMOE_F32: store_as<float, T>(c, blocks, stream); break;
        case BIVMOE_F16: store_as<__half, T>(c, blocks, stream); break;
        default: store_as<__nv_bfloat16, T>(c, blocks, stream);
    }
}

cudaError_t launch_store(const bivmoe_store_args& a, const RopePlan& rope, int ggml_type, int heads, int heads_kv, int head_dim,
                         int page_size, int sm_count, cudaStream_t stream) {
    StoreCall c{a, rope, FastDiv((uint32_t)page_size), heads, heads_kv, head_dim, true};
    const int64_t unit = a.q.ggml_type == BIVMOE_F32 ? 4 : 8;
    for (const bivmoe_rows* r : {&a.q, &a.k, &a.v})
        c.wide = c.wide && (uintptr_t)r->data % 16 == 0 && r->stride_token % unit == 0 && r->stride_head % unit == 0;
    const int blocks = min(a.n_tokens, sm_count * (2048 / kStoreThreads));
    if (ggml_type == BIVMOE_F16) store_from<__half>(c, blocks, stream);
    else store_from<__nv_bfloat16>(c, blocks, stream);
    count_launch();
    return cudaGetLastError();
}

}  // namespace bivmoe
