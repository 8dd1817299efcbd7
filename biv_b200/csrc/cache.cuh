// The paged key/value cache: what its kernels share.  Arguments as the kernels take them, the
// addresses of keys in the pages, which keys a row sees, how a batch of requests is cut into items of
// work on the device, and the careful row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/bivmoe.h"

namespace bivmoe {

constexpr int kCacheSeqs = 1024;            // requests of a call
constexpr int kCacheTokens = 1 << 20;       // new tokens of a call
constexpr int kCachePositions = 1 << 30;    // lengths beyond this are cut here: positions are 32-bit
constexpr int kRopePairs = 128;             // half the widest head

// n / d for 0 <= n < 2^31 by a product: mul = ceil(2^(31 + shift) / d) with 2^shift >= d is at most
// 2^32 - 1 apart from d = 1, and its error, below 2^shift / d <= 1 in 2^(31 + shift), never reaches the
// next quotient.
struct FastDiv {
    uint32_t d = 1, shift = 0;
    uint64_t mul = 1ull << 31;
    FastDiv() = default;
    explicit FastDiv(uint32_t by) : d(by) {
        while ((1ull << shift) < d) shift++;
        mul = ((1ull << (31 + shift)) + d - 1) / d;
    }
    __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return (uint32_t)(((uint64_t)n * mul) >> (31 + shift));
    }
};

struct RopePlan {                    // made when the handle is
    int n_rot, adjacent;
    const double* turns;             // device, [n_rot / 2]: base^(-2i / n_rot) / (2 pi)
    const int32_t* axis;             // device, [n_rot / 2]
};

struct Pool {
    uint8_t* data;
    int64_t page, token, head;       // strides in bytes
    int64_t n_pages;
};

struct AttendCall {
    const uint8_t* q;
    uint8_t* out;
    int64_t q_token, q_head, out_token, out_head;   // strides in bytes
    Pool k, v;
    const int32_t* table;
    int64_t table_stride;
    int table_width, n_seq, n_tokens;
    const int32_t *first, *length;
    FastDiv page, group;             // group: query heads to a kv head
    int heads_kv, window, sinks;
    float scale_log2;                // scale * log2(e): the softmax is taken in powers of two
    float* part_o;                   // [parts][rows][head_dim], not yet divided by the sum
    float2* part_ml;                 // [parts][rows]: running maximum and sum
    int32_t* arrived;                // [parts]: how many parts of a tile are there; zero between calls
    int32_t* status;
    int parts, target;               // room for parts; into how many equal pieces the work is cut at most
};

// ---- requests ------------------------------------------------------------------------------------
// Rows of request b, and what a row sees.  Inconsistent lists (more rows than tokens, a negative
// length) give rows that see less, never an access outside the arrays.
struct Request {
    int begin, rows, past;           // first row (token), rows * group, position of the first row's token
};
__device__ __forceinline__ Request request_of(const AttendCall& a, int b) {
    const int f0 = a.first[b], f1 = a.first[b + 1], len = a.length[b];
    const int lo = max(f0, 0), hi = min(f1, a.n_tokens);
    Request r;
    r.begin = lo;
    r.rows = hi > lo ? (hi - lo) * (int)a.group.d : 0;
    // the last row is the token at len - 1, whatever was cut off
    r.past = max(min(len, kCachePositions), 0) - (f1 - lo);
    return r;
}
// The key tiles that some position from p0 to p1 sees: the first `ns` tiles (the sinks'), then
// consecutive ones from `from` on.
struct TileList {
    int ns, from, n;
    __device__ __forceinline__ int tile(int i) const { return i < ns ? i : i - ns + from; }
};
template <int KT> __device__ __forceinline__ TileList tiles_of(const AttendCall& a, int p0, int p1) {
    TileList t{0, 0, 0};
    if (p1 < 0) return t;
    const int last = p1 / KT;
    if (a.window > 0) {
        const int lo = max(p0, 0) - a.window + 1;
        if (lo > 0) {
            t.from = lo / KT;
            t.ns = min((min(a.sinks, p1 + 1) + KT - 1) / KT, t.from);
        }
    }
    t.n = t.ns + last - t.from + 1;
    return t;
}
// an upper bound of tiles_of().n over the row tiles of a request
template <int KT> __device__ __forceinline__ int most_tiles(const AttendCall& a, const Request& r, int tile_rows) {
    const int tokens = (int)a.group.div(r.rows), p1 = r.past + tokens - 1;
    if (p1 < 0) return 0;
    const int all = p1 / KT + 1;
    if (a.window <= 0) return all;
    const int span = min(tokens, tile_rows / (int)a.group.d + 2);
    const int64_t some = (int64_t)(min(a.sinks, p1 + 1) + KT - 1) / KT + ((int64_t)a.window + span) / KT + 2;
    return some < all ? (int)some : all;
}
__device__ __forceinline__ bool sees(const AttendCall& a, int p, int j) {
    return j <= p && (a.window <= 0 || p - j < a.window || j < a.sinks);
}
// where key j of request b lies: the page, or -1
__device__ __forceinline__ int page_of(const AttendCall& a, const int32_t* row, int j, int& in_page) {
    const uint32_t i = a.page.div((uint32_t)j);
    in_page = j - (int)(i * a.page.d);
    if (i >= (uint32_t)a.table_width) return -1;
    const int page = row[i];
    return page >= 0 && page < a.k.n_pages ? page : -1;
}

// ---- items of work -------------------------------------------------------------------------------
// An item is a tile of TR rows of a request's kv head (row r: token r / group, query head r % group:
// the heads that share keys share the tile) against at most `len` of the key tiles that the tile sees.
// `len` is the same in the whole call: the work in key tiles, W, over `target` pieces, so that the
// parts that have to be joined number at most 2 W / len <= 2 target whatever the lengths are.  Every
// block finds the items by itself from the lengths: it needs no list in memory and no launch before.
struct Items {
    int len, total;
    const int* first_item;           // shared, [n_seq + 1]
    const int* first_part;           // shared, [n_seq + 1]; requests whose tiles are cut only
};
template <int KT, int TR, int THREADS>
__device__ __forceinline__ Items find_items(const AttendCall& a, int least, int* sh /* 2 (n_seq + 1) + THREADS / 16 + 4 */) {
    constexpr int WARPS = THREADS / 32;
    int* first_item = sh;
    int* first_part = sh + a.n_seq + 1;
    int* warps = sh + 2 * (a.n_seq + 1);
    float* works = (float*)(warps + 2 * WARPS);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int each = (a.n_seq + THREADS - 1) / THREADS, b0 = tid * each, b1 = min(b0 + each, a.n_seq);
    // W as a float: it is only what `len` is chosen by, and every block sums it in the same order
    float w = 0.0f;
    for (int b = b0; b < b1; b++) {
        const Request r = request_of(a, b);
        const int nt = (r.rows + TR - 1) / TR, c = nt ? most_tiles<KT>(a, r, TR) : 0;
        first_item[b] = nt;
        first_part[b] = c;
        w += (float)nt * (float)c;
    }
    for (int d = 16; d; d >>= 1) w += __shfl_xor_sync(0xffffffffu, w, d);
    if (lane == 0) works[warp] = w;
    __syncthreads();
    w = 0.0f;
    for (int i = 0; i < WARPS; i++) w += works[i];
    Items it;
    // one more than the quotient: the float's rounding may not make more pieces than there is room for
    it.len = max(least, (int)fminf(w * (float)a.heads_kv / (float)a.target * 1.0001f, 1e9f) + 1);
    int items = 0, parts = 0;
    for (int b = b0; b < b1; b++) {
        const int nt = first_item[b], s = (first_part[b] + it.len - 1) / it.len;
        first_item[b] = items;
        first_part[b] = parts;
        items += nt * a.heads_kv * max(s, 1);
        if (s > 1) parts += nt * a.heads_kv * s;
    }
    int xi = items, xp = parts;
    for (int d = 1; d < 32; d <<= 1) {
        const int yi = __shfl_up_sync(0xffffffffu, xi, d), yp = __shfl_up_sync(0xffffffffu, xp, d);
        if (lane >= d) { xi += yi; xp += yp; }
    }
    if (lane == 31) { warps[2 * warp] = xi; warps[2 * warp + 1] = xp; }
    __syncthreads();
    int bi = xi - items, bp = xp - parts;
    it.total = 0;
    for (int i = 0; i < WARPS; i++) {
        if (i < warp) { bi += warps[2 * i]; bp += warps[2 * i + 1]; }
        it.total += warps[2 * i];
    }
    for (int b = b0; b < b1; b++) { first_item[b] += bi; first_part[b] += bp; }
    if (tid == 0) first_item[a.n_seq] = it.total;
    it.first_item = first_item;
    it.first_part = first_part;
    __syncthreads();
    return it;
}
constexpr size_t items_smem(int n_seq, int threads) {
    return ((2 * ((size_t)n_seq + 1) + 3 * (threads / 32) + 4) * 4 + 15) / 16 * 16;
}
struct Item {
    int b, head, row0, rows;         // request, kv head, the tile's first row and how many of its rows there are
    Request r;
    TileList tiles;
    int i0, i1;                      // of the tile list
    int split, splits, part;         // which piece of how many; the first piece's place among the parts
};
// Long tiles first: within a request the last rows see the most.
template <int KT, int TR> __device__ __forceinline__ Item item_at(const AttendCall& a, const Items& it, int index) {
    int lo = 0, hi = a.n_seq;        // the request: the last one that begins at or before the item
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (it.first_item[mid] <= index) lo = mid; else hi = mid;
    }
    Item x;
    x.b = lo;
    x.r = request_of(a, lo);
    const int nt = (x.r.rows + TR - 1) / TR;
    const int most = max((most_tiles<KT>(a, x.r, TR) + it.len - 1) / it.len, 1);
    int rest = index - it.first_item[lo];
    x.split = rest % most;
    rest /= most;
    x.head = rest % a.heads_kv;
    const int t = nt - 1 - rest / a.heads_kv;
    x.row0 = t * TR;
    x.rows = min(TR, x.r.rows - x.row0);
    const int p0 = x.r.past + (int)a.group.div(x.row0), p1 = x.r.past + (int)a.group.div(x.row0 + x.rows - 1);
    x.tiles = tiles_of<KT>(a, p0, p1);
    x.i0 = x.split * it.len;
    x.i1 = min(x.i0 + it.len, x.tiles.n);
    x.splits = (x.tiles.n + it.len - 1) / it.len;
    x.part = it.first_part[lo] + (t * a.heads_kv + x.head) * most;
    return x;
}
// what a piece beyond the tile's own number of pieces has to do: nothing; the first one of a tile
// that sees nothing writes its zeros
__device__ __forceinline__ bool item_void(const Item& x) { return x.split > 0 && x.i0 >= x.i1; }

// ---- types ---------------------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <class T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- the careful row -------------------------------------------------------------------------------
// A weight of zero times an infinity or a NaN is a NaN, so in the tiled products a value that a row does
// not see could reach it.  Rows that come out of them not finite are computed again like this, by a warp,
// from the keys that they see alone; a row that does see such values has its NaN after the first of
// them.  Lane l holds the values l, l + 32, ... of o.
template <int D, class T>
__device__ __noinline__ void careful_row(const AttendCall& a, const Item& x, int row, int kt, float (&o)[D / 32], float& m, float& l) {
    const int lane = threadIdx.x & 31, R = x.row0 + row;
    const int tok = (int)a.group.div(R), h = x.head * (int)a.group.d + R - tok * (int)a.group.d, p = x.r.past + tok;
    const T* q = (const T*)(a.q + (int64_t)(x.r.begin + tok) * a.q_token + (int64_t)h * a.q_head);
    const int32_t* table = a.table + (int64_t)x.b * a.table_stride;
    float qv[D / 32];
    for (int i = 0; i < D / 32; i++) { qv[i] = to_f32(q[lane + 32 * i]); o[i] = 0.0f; }
    m = -INFINITY;
    l = 0.0f;
    for (int i = x.i0; i < x.i1; i++) {
        const int j0 = x.tiles.tile(i) * kt;
        for (int j = j0; j < j0 + kt && j <= p; j++) {
            int at;
            const int page = sees(a, p, j) ? page_of(a, table, j, at) : -1;
            if (page < 0) continue;
            const T* k = (const T*)(a.k.data + page * a.k.page + at * a.k.token + x.head * a.k.head);
            const T* v = (const T*)(a.v.data + page * a.v.page + at * a.v.token + x.head * a.v.head);
            float s = 0.0f;
            for (int e = 0; e < D / 32; e++) s += qv[e] * to_f32(k[lane + 32 * e]);
            for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            s *= a.scale_log2;
            const float mn = fmaxf(m, s), c = mn == -INFINITY ? 1.0f : exp2_of(m - mn), e2 = mn == -INFINITY ? 0.0f : exp2_of(s - mn);
            if (s != s || mn == INFINITY) {       // the softmax of a NaN, or of infinity: NaN
                for (int e = 0; e < D / 32; e++) o[e] = NAN;
                l = NAN;
                return;
            }
            m = mn;
            l = l * c + e2;
            for (int e = 0; e < D / 32; e++) o[e] = o[e] * c + e2 * to_f32(v[lane + 32 * e]);
        }
    }
}

size_t attend_few_smem(int head_dim, int n_seq);
cudaError_t launch_attend_few(const AttendCall& a, int head_dim, int ggml_type, int sm_count, cudaStream_t stream);
cudaError_t launch_extend(const bivmoe_extend_args& a, int page_size, int sm_count, cudaStream_t stream);
cudaError_t launch_store(const bivmoe_store_args& a, const RopePlan& rope, int ggml_type, int heads, int heads_kv, int head_dim,
                         int page_size, int sm_count, cudaStream_t stream);
// the rows, and the pieces of work, that the workspace is sized for
constexpr int kFewRows = 16;

}  // namespace bivmoe
