// The paged key/value cache: what its kernels share.  Arguments as the kernels take them, the
// addresses of keys in the pages, which keys a row sees, how the work of a batch is shared out on the
// device, and the careful row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/bivmoe.h"

namespace bivmoe {

constexpr int kCacheSeqs = 1024;            // requests of a call
constexpr int kCacheTokens = 1 << 20;       // new tokens of a call
constexpr int kCachePositions = 1 << 29;    // lengths beyond this are cut here: sums of two positions and a window are 32-bit
constexpr int kCachePages = 1 << 20;        // new pages of a request and call
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
    float* part_o;                   // [2 blocks][rows][head_dim], not yet divided by the sum
    float2* part_ml;                 // [2 blocks][rows]: running maximum and sum
    int32_t* arrived;                // [blocks][..]: how many pieces of a tile are there; zero between calls
    int32_t* status;
};

// ---- requests ------------------------------------------------------------------------------------
// Rows of request b, and what a row sees.  Inconsistent lists (more rows than tokens, a negative
// length) give rows that see less, never an access outside the arrays.
struct Request {
    int begin, rows, past;           // first row (token), rows * group, position of the first row's token
};
__host__ __device__ __forceinline__ Request request_of(const AttendCall& a, int b) {
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
    __host__ __device__ __forceinline__ int tile(int i) const { return i < ns ? i : i - ns + from; }
};
template <int KT> __host__ __device__ __forceinline__ TileList tiles_of(const AttendCall& a, int p0, int p1) {
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
// whether some row from p0 to p1 sees key j
__device__ __forceinline__ bool seen(const AttendCall& a, int p0, int p1, int j) {
    return j <= p1 && (a.window <= 0 || j > p0 - a.window || j < a.sinks);
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

// ---- shares of the work ----------------------------------------------------------------------------
// A tile is TR rows of a request's kv head (row r: token r / group, query head r % group: the heads that
// share keys share the tile); its work is the key tiles it sees, one unit each (a tile that sees none:
// one, for its zeros), and EXTRA units before them that stand for what a tile costs besides (its rows
// in, its sums out).  The units of all tiles stand in one line, requests, kv heads, tiles, key tiles
// in this order, and each of `g` blocks takes an equal share of the line, wherever that cuts a tile:
// the blocks end together whatever the lengths are, and a block has at most two pieces of tiles
// that others share, so that the room for pieces is two to a block.  Every block finds its share by
// itself from the lengths: no list in memory, no launch before.
// a / b for a >= 0, b > 0; most are short
__host__ __device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (a | b) >> 31 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
// (the shares' arithmetic is tested on the host, where the block is this one)
inline int& host_block() {
    static thread_local int block = 0;
    return block;
}
struct Share {
    int64_t lo, hi;                  // this block's units
    int64_t each, longer;            // units of a block; those of the first blocks, which have one more
    const int64_t* before;           // shared, [n_seq + 1]: units of the requests before
    __host__ __device__ __forceinline__ int block() const {
#ifdef __CUDA_ARCH__
        return (int)blockIdx.x;
#else
        return host_block();
#endif
    }
    // this block's of `units`, of which `least` are worth a block, shared out over up to `blocks`
    __host__ __device__ __forceinline__ void take(int64_t units, int least, int blocks) {
        const int64_t worth = quotient(units + least - 1, least);
        const int g = (int)(worth < blocks ? worth : blocks), c = block();
        lo = hi = each = longer = 0;
        if (c >= g) return;
        each = quotient(units, g);
        const int more = (int)(units - each * g);
        longer = more * (each + 1);
        lo = each * c + min(c, more);
        hi = lo + each + (c < more);
    }
    // the block that has unit u
    __host__ __device__ __forceinline__ int owner(int64_t u) const {
        return u < longer ? (int)quotient(u, each + 1) : (int)(quotient(longer, each + 1) + quotient(u - longer, each));
    }
};
template <int KT, int TR> __host__ __device__ __forceinline__ TileList tile_list(const AttendCall& a, const Request& r, int t) {
    return tiles_of<KT>(a, r.past + (int)a.group.div(t * TR), r.past + (int)a.group.div(min((t + 1) * TR, r.rows) - 1));
}
template <int KT, int TR, int EXTRA> __host__ __device__ __forceinline__ int tile_units(const AttendCall& a, const Request& r, int t) {
    return EXTRA + max(tile_list<KT, TR>(a, r, t).n, 1);
}
constexpr size_t share_smem(int n_seq, int threads) { return (((size_t)n_seq + 1 + threads / 32) * 8 + 15) / 16 * 16; }
constexpr int kAlone = 4;            // tiles of a request that one thread counts
// least: units that are worth a block
template <int KT, int TR, int EXTRA, int THREADS>
__device__ __forceinline__ Share find_share(const AttendCall& a, int least, int64_t* sh /* share_smem */) {
    constexpr int WARPS = THREADS / 32;
    int64_t* before = sh;
    int64_t* sums = sh + a.n_seq + 1;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t carry = 0;
    for (int b0 = 0; b0 < a.n_seq; b0 += THREADS) {
        const int b = b0 + tid;
        Request r{0, 0, 0};
        if (b < a.n_seq) r = request_of(a, b);
        const int nt = (r.rows + TR - 1) / TR;
        int64_t units = 0;
        if (nt <= kAlone)
            for (int t = 0; t < nt; t++) units += tile_units<KT, TR, EXTRA>(a, r, t);
        for (uint32_t many = __ballot_sync(0xffffffffu, nt > kAlone); many; many &= many - 1) {
            const int of = __ffs(many) - 1;   // a long one: counted by the warp
            const Request q{__shfl_sync(0xffffffffu, r.begin, of), __shfl_sync(0xffffffffu, r.rows, of), __shfl_sync(0xffffffffu, r.past, of)};
            int64_t some = 0;
            for (int t = lane; t < (q.rows + TR - 1) / TR; t += 32) some += tile_units<KT, TR, EXTRA>(a, q, t);
            for (int d = 16; d; d >>= 1) some += __shfl_xor_sync(0xffffffffu, some, d);
            if (lane == of) units = some;
        }
        units *= a.heads_kv;
        int64_t x = units;
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        int64_t base = carry;
        for (int i = 0; i < WARPS; i++) {
            if (i < warp) base += sums[i];
            carry += sums[i];
        }
        if (b < a.n_seq) before[b] = base + x - units;
    }
    if (tid == 0) before[a.n_seq] = carry;
    __syncthreads();
    Share s;
    s.before = before;
    s.take(carry, least, (int)gridDim.x);
    return s;
}
struct Piece {
    int b, head, row0, rows;         // request, kv head, the tile's first row and how many of its rows there are
    Request r;
    TileList tiles;
    int i0, n;                       // first of the tile list, and how many
    int part, parts;                 // which piece of how many
    int c0;                          // the block that has the first one
    // where a piece's unfinished sums stand: a block is the first of at most one cut tile, and has
    // at most one piece of a tile that began before it
    __host__ __device__ __forceinline__ int slot(int p) const { return p == 0 ? 2 * c0 + 1 : 2 * (c0 + p); }
};
// The pieces of a block's share, one after another: every warp goes through them by itself.
// A share's end that lies at most SNAP units behind a tile's beginning, or before its end, is moved there:
// a tile that is cut costs its unfinished sums' way out and in (SNAP >= EXTRA: no piece is without keys).
template <int KT, int TR, int EXTRA, int SNAP> struct Walk {
    static_assert(SNAP >= EXTRA, "");
    const AttendCall& a;
    const Share& s;
    int64_t at;                      // the next unit
    int b, head, t, nt, off;         // where it lies: of which tile, and how far in
    Request r;
    __host__ __device__ __forceinline__ Walk(const AttendCall& call, const Share& share) : a(call), s(share), at(share.lo) {
        if (at >= s.hi) return;
        int lo = 0, hi = a.n_seq;    // the request: the last one that begins at or before the unit
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s.before[mid] <= at) lo = mid; else hi = mid;
        }
        open(lo);
        const int64_t rest = at - s.before[b], each = quotient(s.before[b + 1] - s.before[b], a.heads_kv);
        head = (int)quotient(rest, each);
        int64_t in = rest - head * each;
        find_tile(in);
        off = (int)in;
        const int units = tile_units<KT, TR, EXTRA>(a, r, t);
        if (off <= SNAP) {
            at -= off;
            off = 0;
        } else if (units - off <= SNAP) {
            at += units - off;
            step();
        }
    }
    // t: the tile that has unit `in` of its request's head, and which of its own units that is
    __host__ __device__ __forceinline__ void find_tile(int64_t& in) {
        t = 0;
#ifdef __CUDA_ARCH__
        const int lane = threadIdx.x & 31;
        while (nt > 1 && t < nt) {   // 32 of them at a time
            const int mine = t + lane < nt ? tile_units<KT, TR, EXTRA>(a, r, t + lane) : 0;
            int64_t x = mine;
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
                if (lane >= d) x += y;
            }
            const uint32_t beyond = __ballot_sync(0xffffffffu, x > in);
            if (beyond) {
                const int of = __ffs(beyond) - 1;
                in -= __shfl_sync(0xffffffffu, x - mine, of);
                t += of;
                break;
            }
            in -= __shfl_sync(0xffffffffu, x, 31);
            t += 32;
        }
#else
        for (int u; nt > 1 && in >= (u = tile_units<KT, TR, EXTRA>(a, r, t)); t++) in -= u;
#endif
    }
    __host__ __device__ __forceinline__ void open(int request) {
        b = request;
        r = request_of(a, b);
        nt = (r.rows + TR - 1) / TR;
    }
    // to the beginning of the tile that follows, at `at`
    __host__ __device__ __forceinline__ void step() {
        off = 0;
        if (++t < nt) return;
        t = 0;
        if (++head < a.heads_kv) return;
        head = 0;
        if (at >= s.before[a.n_seq]) return;
        int next = b + 1;
        while (s.before[next + 1] == s.before[next]) next++;   // those without rows
        open(next);
    }
    // The next piece; false at the share's end.
    __host__ __device__ __forceinline__ bool next(Piece& x) {
        if (at >= s.hi) return false;
        x.tiles = tile_list<KT, TR>(a, r, t);
        const int units = EXTRA + max(x.tiles.n, 1);
        const int64_t u0 = at - off;
        int end = units;
        if (s.hi - u0 < units) {
            const int e = (int)(s.hi - u0);
            if (e <= SNAP) {
                at = s.hi;
                return false;
            }
            if (units - e > SNAP) end = e;
        }
        x.b = b;
        x.head = head;
        x.r = r;
        x.row0 = t * TR;
        x.rows = min(TR, r.rows - x.row0);
        x.i0 = max(off - EXTRA, 0);
        x.n = min(end - EXTRA, x.tiles.n) - x.i0;
        x.part = 0;
        x.parts = 1;
        x.c0 = s.block();
        if (off > 0 || end < units) {
            x.c0 = s.owner(u0 + SNAP);
            x.parts = s.owner(u0 + units - SNAP - 1) - x.c0 + 1;
            x.part = s.block() - x.c0;
        }
        at = u0 + end;
        off = end;
        if (end == units) step();
        return true;
    }
};

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
// 16 bytes into shared memory, under way until the thread waits for it: nothing is read, and zeros are
// written, where there is nothing
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// The powers of two by which the weights that go into the second product are lifted above one.
// f16 keeps its 11 bits down to 2^-14 and nothing below 2^-25, and the many small weights beside one large key
// count together: up to 2^15.  bf16 has f32's exponents, and so have its values: weights of at most 2^-24 keep
// the sums over up to 2^24 keys in f32 whatever the values are, where the weights' sum is yet to be divided by.
// The maximum that a piece is written with is lowered by as much, so that pieces join as they are.
template <class T> __device__ __forceinline__ constexpr float weight_lift() { return -24.0f; }
template <> __device__ __forceinline__ constexpr float weight_lift<__half>() { return 15.0f; }

// ---- the careful row -------------------------------------------------------------------------------
// A weight of zero times an infinity or a NaN is a NaN, so in the tiled products a value that a row does
// not see could reach it.  A row that comes out of them not finite is asked whether it has met such a
// value; if not, what it sees has made it what it is, and it stays.  If it has, it is computed again, by
// a warp, from the keys that it sees alone.  A value that a row does see reaches it whatever its weight,
// and a piece of a weight that is zero in f32 takes part in the join for that: which keys share a piece is
// not the row's matter.
// Eight requests of 100000 tokens, 256 of them new, 16 / 4 heads of 128: 1.77 ms; with an early infinity
// that all rows see 1.87; with a NaN in one request's last token, which 255 of its 256 rows have to be kept
// from, 633 (7 us a row and 32 keys: a trip to memory for the keys, four for the values).

// Two values of T, and whether they are finite: 0, or NaN.
template <class T> __device__ __forceinline__ float2 both(uint32_t w) {
    const T* e = (const T*)&w;
    return make_float2(to_f32(e[0]), to_f32(e[1]));
}

// Whether row `row` has met a value that it does not see and that is not finite: in the key tiles (of kt
// keys) that are hidden from it in part, among the keys up to the rows' last one, beyond which nothing is
// fetched.  For a whole warp.
template <int D, class T>
__device__ __noinline__ bool met_hidden(const AttendCall& a, const Piece& x, int row, int kt) {
    const int lane = threadIdx.x & 31, p = x.r.past + (int)a.group.div(x.row0 + row), top = x.r.past + (int)a.group.div(x.row0 + x.rows - 1);
    const int32_t* table = a.table + (int64_t)x.b * a.table_stride;
    for (int i0 = 0; i0 < x.n; i0 += 32) {
        const int i = i0 + lane, j0 = i < x.n ? x.tiles.tile(x.i0 + i) * kt : 0;
        const bool whole = i >= x.n || (j0 + kt - 1 <= p && (a.window <= 0 || p - j0 < a.window || j0 + kt <= a.sinks));
        for (uint32_t partly = __ballot_sync(0xffffffffu, !whole); partly; partly &= partly - 1) {
            const int first = __shfl_sync(0xffffffffu, j0, __ffs(partly) - 1);
            float odd = 0.0f;                     // NaN as soon as something is not finite
            for (int j = first + lane; j < first + kt; j += 32) {
                int at;
                const int page = j <= top && !sees(a, p, j) ? page_of(a, table, j, at) : -1;
                if (page < 0) continue;
                const uint4* v = (const uint4*)(a.v.data + page * a.v.page + at * a.v.token + x.head * a.v.head);
#pragma unroll 8
                for (int c = 0; c < D / 8; c++) {
                    const uint4 w = v[c];
                    for (const uint32_t u : {w.x, w.y, w.z, w.w}) {
                        const float2 y = both<T>(u);
                        odd = fmaf(y.x, 0.0f, fmaf(y.y, 0.0f, odd));
                    }
                }
            }
            if (__any_sync(0xffffffffu, odd != 0.0f)) return true;
        }
    }
    return false;
}

// The row again, 32 keys at a time, a lane to a key for the scores; then lane l holds the values l, l + 32,
// ... of o, and all 32 keys' loads are under way together.  A row that sees a score of NaN or infinity ends
// there, as a piece that every join gives the weight 1 (maximum -infinity, sum NaN).
template <int D, class T>
__device__ __noinline__ void careful_row(const AttendCall& a, const Piece& x, int row, int kt, float (&o_out)[D / 32], float& m_out, float& l_out) {
    const int lane = threadIdx.x & 31, R = x.row0 + row;
    const int tok = (int)a.group.div(R), h = x.head * (int)a.group.d + R - tok * (int)a.group.d, p = x.r.past + tok;
    const uint4* q = (const uint4*)(a.q + (int64_t)(x.r.begin + tok) * a.q_token + (int64_t)h * a.q_head);
    const uint8_t *keys = a.k.data + x.head * a.k.head, *values = a.v.data + x.head * a.v.head;
    const int32_t* table = a.table + (int64_t)x.b * a.table_stride;
    // (of its own, not the caller's in memory: a store there would keep the next key's loads from going ahead of it)
    float o[D / 32] = {}, m = -INFINITY, l = 0.0f;
    for (int i = x.i0; i < x.i0 + x.n; i++) {
        const int j0 = x.tiles.tile(i) * kt;
        for (int j = j0 + lane; j - lane < j0 + kt; j += 32) {
            int at = 0;
            const int page = sees(a, p, j) ? page_of(a, table, j, at) : -1;
            if (!__any_sync(0xffffffffu, page >= 0)) continue;
            float s = -INFINITY;
            if (page >= 0) {
                const uint4* k = (const uint4*)(keys + page * a.k.page + at * a.k.token);
                float d[4] = {};
#pragma unroll 8
                for (int c = 0; c < D / 8; c++) {
                    const uint4 u = q[c], w = k[c];
                    const uint32_t uu[4] = {u.x, u.y, u.z, u.w}, ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float2 f = both<T>(uu[e]), g = both<T>(ww[e]);
                        d[e] = fmaf(f.x, g.x, fmaf(f.y, g.y, d[e]));
                    }
                }
                s = ((d[0] + d[1]) + (d[2] + d[3])) * a.scale_log2;
            }
            if (__any_sync(0xffffffffu, s != s || s == INFINITY)) {       // the softmax of a NaN, or of infinity: NaN
                for (int e = 0; e < D / 32; e++) o_out[e] = NAN;
                l_out = NAN;
                m_out = -INFINITY;
                return;
            }
            float mn = s;
            for (int d = 16; d; d >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
            mn = fmaxf(m, mn);
            const float c = mn == -INFINITY ? 1.0f : exp2_of(m - mn), e2 = mn == -INFINITY ? 0.0f : exp2_of(s - mn + weight_lift<T>());
            float sum = e2;
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            m = mn;
            l = l * c + sum;
#pragma unroll
            for (int e = 0; e < D / 32; e++) o[e] *= c;
            const int64_t place = page >= 0 ? page * a.v.page + at * a.v.token : -1;
#pragma unroll 8
            for (int t = 0; t < 32; t++) {
                const int64_t of = __shfl_sync(0xffffffffu, place, t);
                const float w = __shfl_sync(0xffffffffu, e2, t);
                const T* v = (const T*)(values + max(of, (int64_t)0)) + lane;      // (some page is there: so is the first)
#pragma unroll
                for (int e = 0; e < D / 32; e++) {
                    const float y = to_f32(v[32 * e]);
                    o[e] = of >= 0 ? fmaf(w, y, o[e]) : o[e];
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < D / 32; e++) o_out[e] = o[e];
    m_out = m - weight_lift<T>();
    l_out = l;
}

cudaError_t launch_attend_few(const AttendCall& a, int head_dim, int ggml_type, int sm_count, cudaStream_t stream);
cudaError_t launch_attend_tc(const AttendCall& a, int head_dim, int ggml_type, int sm_count, cudaStream_t stream);
cudaError_t launch_extend(const bivmoe_extend_args& a, int page_size, unsigned long long* unstored, int sm_count, cudaStream_t stream);
cudaError_t launch_store(const bivmoe_store_args& a, const RopePlan& rope, int ggml_type, int heads, int heads_kv, int head_dim,
                         int page_size, int sm_count, cudaStream_t stream);
// what the workspace is sized for: rows of a tile, blocks to a multiprocessor
constexpr int kFewRows = 16;
// (heads of 64, a windowed step of 128 requests: two blocks 75.1, three 69.7, four of 128 registers 70.0 us)
constexpr int few_blocks(int head_dim) { return head_dim == 256 ? 1 : head_dim == 128 ? 2 : 3; }
constexpr int tc_rows(int head_dim) { return head_dim == 256 ? 128 : 256; }

}  // namespace bivmoe
