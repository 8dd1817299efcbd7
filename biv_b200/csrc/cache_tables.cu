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
// Bound by latency: launch, one load, the sums, one search, one load: 64 requests of a token each 3.2 us,
// 1000 requests with 30880 rows 5.1.
constexpr int kExtendThreads = 256;
constexpr int kExtendEach = kCacheSeqs / kExtendThreads;

struct ExtendCall {
    bivmoe_extend_args a;
    FastDiv page;
    unsigned long long* unstored;    // of the handle: new tokens without a slot so far
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
    pdl_enter();
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
            need[i] = min(max((int)c.page.div(past + add[i] + c.page.d - 1) - have, 0), kCachePages);
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
    int lost = me == 0 ? max(all_t - a.n_tokens, 0) : 0;
    for (int t = me; t < a.n_tokens; t += step) {
        int64_t slot = -1;
        int p = 0;
        if (t < all_t) {
            const int b = last_at_or_before(s_first, n, t);
            p = s_past[b] + t - s_first[b];
            const int at = (int)c.page.div(p);
            if (at < a.table_width) {
                const int i = s_page[b] + at - s_have[b];   // of the new pages
                const bool given = i < min(count, s_page[b + 1]);
                const int page = at < s_have[b] ? a.table[b * a.table_stride + at] : given ? a.free_pages[count - 1 - i] : -1;
                if (page >= 0) slot = (int64_t)page * c.page.d + (p - at * (int)c.page.d);
            }
            lost += slot < 0;
        }
        a.slots[t] = slot;
        a.positions[t] = p;
    }
    lost = __reduce_add_sync(0xffffffffu, lost);
    if (lane == 0 && lost) atomicAdd(c.unstored, (unsigned long long)lost);
}

cudaError_t launch_extend(const bivmoe_extend_args& a, int page_size, unsigned long long* unstored, int sm_count, cudaStream_t stream) {
    ExtendCall c{a, FastDiv((uint32_t)page_size), unstored};
    // a few rows a thread: more blocks only repeat the sums
    const int blocks = (int)min((int64_t)sm_count, ((int64_t)a.n_tokens + 2 * kExtendThreads - 1) / (2 * kExtendThreads) + 1);
    count_launch();
    return launch_with(pdl_mode() != 0, stream, extend_kernel, dim3(blocks), dim3(kExtendThreads), 0, c);
}

// ---- store ---------------------------------------------------------------------------------------
// (x, y) -> (x cos t - y sin t, x sin t + y cos t) for the pairs of the head's first n_rot values, t the
// token's position on the pair's axis times base^(-2i / n_rot).  A position times a frequency loses
// whole radians in f32 long before a cache is full (2^18 tokens: 0.01 rad), so the angle is made in
// f64, in turns, its whole turns taken off, and only the rest goes to f32 for the sine and cosine,
// once for each token and pair of a warp's heads.
// Bound by memory: a row is read once and written once, in 16-byte pieces.  A warp takes a token (of few
// tokens, some of a token's heads).  A lane keeps to 16 values of the head, whatever the head: the
// lanes of one such column make its sines between them and pass them round, so that nothing is shared
// beyond the warp.  What hides a row's way from memory is the number of warps: with the values of one
// round of heads to a thread (64 registers, 32 warps an SM) 16381 tokens of 32 + 8 + 8 heads of 128 take
// 75 us, 403 MB at 5.4 TB/s; with two rounds 87, with four (16 warps) 101; a block to a token 152.  Rows of f32 93 us, 604 MB at 6.5 TB/s.
constexpr int kStoreWarps = 4;

struct StoreCall {
    bivmoe_store_args a;
    RopePlan rope;
    FastDiv page;
    int heads, heads_kv;
    int parts;                       // warps to a token
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
template <class In, class T, bool ADJACENT, int D>
__global__ void __launch_bounds__(32 * kStoreWarps, 8) store_kernel(const __grid_constant__ StoreCall c) {
    constexpr int COLUMNS = D / 16, ROWS = 32 / COLUMNS, OWN = 8 / ROWS;   // units of a head, heads at once, pairs a lane makes
    const bivmoe_store_args& a = c.a;
    pdl_enter();
    const int lane = threadIdx.x & 31, job = blockIdx.x * kStoreWarps + (threadIdx.x >> 5);
    const int t = job / c.parts, part = job - t * c.parts;
    if (t >= a.n_tokens) return;
    const int col = lane % COLUMNS, sub = lane / COLUMNS, rows = c.heads + 2 * c.heads_kv;
    const int rounds = (rows + ROWS - 1) / ROWS, r0 = rounds * part / c.parts, r1 = rounds * (part + 1) / c.parts;
    const int pairs = c.rope.n_rot / 2;
    const bool turns = col < c.rope.n_rot / 16;
    const int turned_at = ADJACENT ? 16 * col : 8 * col, turned_gap = ADJACENT ? 8 : pairs;
    const int64_t slot = a.slots[t];              // (one past 2^31 is past any pool that fits the device)
    const int64_t page = slot >= 0 && slot >> 31 == 0 ? (int64_t)c.page.div((uint32_t)slot) : -1;
    const int at = (int)(slot - page * c.page.d);
    const bool kept = page >= 0 && page < a.k_pool.n_pages && page < a.v_pool.n_pages;
    float co[8], si[8];
    for (int r = r0; r < r1; r++) {
        const int row = r * ROWS + sub;
        const bool is_q = row < c.heads, is_k = !is_q && row < c.heads + c.heads_kv, turn = turns && (is_q || is_k);
        const int h = is_q ? row : is_k ? row - c.heads : row - c.heads - c.heads_kv;
        const int off = turn ? turned_at : 16 * col, gap = turn ? turned_gap : 8;
        float x[8], y[8];
        if (row < rows) {
            const bivmoe_rows& in = is_q ? a.q : is_k ? a.k : a.v;
            const In* from = (const In*)in.data + t * in.stride_token + h * in.stride_head + off;
            load8(from, c.wide, x);
            load8(from + gap, c.wide, y);
        }
        if (r == r0 && pairs) {
            float own_co[OWN], own_si[OWN];
#pragma unroll
            for (int i = 0; i < OWN; i++) {
                const int pair = 8 * col + sub * OWN + i;
                own_co[i] = 1.0f;
                own_si[i] = 0.0f;
                if (turns) {
                    const double by = (double)a.positions[c.rope.axis[pair] * a.positions_stride + t] * c.rope.turns[pair];
                    sincospif((float)(2.0 * (by - rint(by))), &own_si[i], &own_co[i]);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                co[e] = __shfl_sync(0xffffffffu, own_co[e % OWN], e / OWN * COLUMNS + col);
                si[e] = __shfl_sync(0xffffffffu, own_si[e % OWN], e / OWN * COLUMNS + col);
            }
        }
        if (row >= rows || (!is_q && !kept)) continue;
        if (turn) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float& u = ADJACENT ? (e < 4 ? x[2 * e % 8] : y[2 * e % 8]) : x[e];
                float& v = ADJACENT ? (e < 4 ? x[2 * e % 8 + 1] : y[2 * e % 8 + 1]) : y[e];
                const float p = u * co[e] - v * si[e], q = u * si[e] + v * co[e];
                u = p;
                v = q;
            }
        }
        const bivmoe_pool& pool = is_k ? a.k_pool : a.v_pool;
        T* to = (is_q ? (T*)a.q_out.data + t * a.q_out.stride_token + h * a.q_out.stride_head
                      : (T*)pool.data + page * pool.stride_page + at * pool.stride_token + h * pool.stride_head) + off;
        store8(to, x);
        store8(to + gap, y);
    }
}

template <class In, class T, bool ADJACENT> static cudaError_t store_of(const StoreCall& c, int dim, int blocks, cudaStream_t stream) {
    auto launch = [&](void (*kernel)(StoreCall)) {
        return launch_with(pdl_mode() != 0, stream, kernel, dim3(blocks), dim3(32 * kStoreWarps), 0, c);
    };
    return dim == 64 ? launch(store_kernel<In, T, ADJACENT, 64>)
                     : dim == 128 ? launch(store_kernel<In, T, ADJACENT, 128>) : launch(store_kernel<In, T, ADJACENT, 256>);
}
template <class In, class T> static cudaError_t store_as(const StoreCall& c, int dim, int blocks, cudaStream_t stream) {
    return c.rope.adjacent ? store_of<In, T, true>(c, dim, blocks, stream) : store_of<In, T, false>(c, dim, blocks, stream);
}
template <class T> static cudaError_t store_from(const StoreCall& c, int dim, int blocks, cudaStream_t stream) {
    switch (c.a.q.ggml_type) {
        case BIVMOE_F32: return store_as<float, T>(c, dim, blocks, stream);
        case BIVMOE_F16: return store_as<__half, T>(c, dim, blocks, stream);
        default: return store_as<__nv_bfloat16, T>(c, dim, blocks, stream);
    }
}

cudaError_t launch_store(const bivmoe_store_args& a, const RopePlan& rope, int ggml_type, int heads, int heads_kv, int head_dim,
                         int page_size, int sm_count, cudaStream_t stream) {
    StoreCall c{a, rope, FastDiv((uint32_t)page_size), heads, heads_kv, 1, true};
    const int64_t unit = a.q.ggml_type == BIVMOE_F32 ? 4 : 8;
    for (const bivmoe_rows* r : {&a.q, &a.k, &a.v})
        c.wide = c.wide && (uintptr_t)r->data % 16 == 0 && r->stride_token % unit == 0 && r->stride_head % unit == 0;
    // as many warps to a token as fill the device, at most one for each round of heads
    const int rounds = (heads + 2 * heads_kv + 512 / head_dim - 1) / (512 / head_dim);
    c.parts = max(1, min(rounds, 16 * sm_count / a.n_tokens));
    const int blocks = (int)(((int64_t)a.n_tokens * c.parts + kStoreWarps - 1) / kStoreWarps);
    count_launch();
    return ggml_type == BIVMOE_F16 ? store_from<__half>(c, head_dim, blocks, stream) : store_from<__nv_bfloat16>(c, head_dim, blocks, stream);
}

}  // namespace bivmoe
