// Attention over the pages for tiles of 16 rows: one pass over the keys with the running maximum and
// sum of the softmax, products on the warp-level tensor cores.
//
//   s_j = scale q . k_j,  m = max s_j,  l = sum 2^(s_j - m),  o = sum 2^(s_j - m) v_j / l   (s in powers of two)
//
// A block is four warps; of a tile of 64 keys a warp takes a quarter, in a ring of its own in shared memory
// that its own cp.async copies fill, with its own running maximum, sum and o: the warps meet at the
// piece's end only, where the four o are joined.  The work is shared out over blocks wherever that cuts a
// long axis (cache.cuh); the block that is last to finish a tile joins its pieces, in their own order
// whoever is last.
// With one new token a request the keys are read once, and a batch is bound by memory: 64 requests of 1 to
// 8192 tokens, 32 / 8 heads of 128 (1.1 GB), 185 us, 5.9 TB/s where a copy reaches 6.55.  A single request is
// bound by the chain of trips to memory (lengths, table, keys, pieces out and in) and by the fetch of
// instructions: one token at 1000, 16 / 2 heads of 256, 11.6 us.
#include "cache.cuh"
#include "common.cuh"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace bivmoe {

constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps, kFewStages = 3;
// Key tiles that are worth a block; that a tile costs besides, and that are not worth a cut.  us with 0 / 1 / 2 / 3 of
// the latter: one token at 1000, heads of 256, 11.8 / 12.3 / 14.5 / 15.2, heads of 128 13.0 / 11.6 / 12.9 / 13.5; a
// windowed step of 128 requests 70.2 / 69.8 / 70.5 / 72.2.
constexpr int kFewLeast = 2, kFewExtra = 1;

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <class T> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D> struct Few {
    static constexpr int keys = 16, tile = keys * kFewWarps;
    static constexpr int half = keys * D * 2, stage = 2 * half;   // bytes: k, then v
    static constexpr int ring = kFewWarps * kFewStages * stage;
    static constexpr int fixed = ring + 16 * D * 2;               // and the 16 rows of q
    static constexpr int part = D + 8;                            // floats from row to row where the warps' o meet: 8 rows apart, no bank twice
    static_assert(16 * part * 4 <= kFewStages * stage, "");
};

// bytes from a head's first page on to a key's k and v
struct alignas(16) Place { int64_t k, v; };
// 16-byte piece `c` of row `r`: the low three bits of the piece's place are turned by the row, so that
// eight rows' pieces c lie in different banks
template <int D> __device__ __forceinline__ uint32_t few_at(int r, int c) {
    return (uint32_t)(r * (D * 2) + ((c ^ (r & 7)) << 4));
}

// The pieces of a tile, joined in their order by the block that was last.  The threads divide up the rows
// that there are; four pieces are under way at a time.
template <int D, class T> __device__ __forceinline__ void join(const AttendCall& a, const Piece& x) {
    constexpr int CK = D / 32 < 4 ? D / 32 : 4;   // 16-byte pieces of a row that a thread has under way
    const int per_row = min(kFewThreads / (x.rows > 8 ? 16 : x.rows > 4 ? 8 : 4), D / 4);
    const int row = threadIdx.x / per_row, sub = threadIdx.x - row * per_row;
    if (row >= x.rows) return;
    const int R = x.row0 + row, tok = (int)a.group.div(R), h = x.head * (int)a.group.d + R - tok * (int)a.group.d;
    auto weight = [](float2 ml, float top) {      // a NaN piece has a sum that is one, whatever its maximum
        return ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : exp2_of(ml.x - top);
    };
    for (int c0 = sub * 4; c0 < D; c0 += CK * 4 * per_row) {
        float M = -INFINITY, L = 0.0f;
        float4 y[CK] = {};
#pragma unroll 1
        for (int s0 = 0; s0 < x.parts; s0 += 4) {
            float2 ml[4];
            float4 v[4][CK];
#pragma unroll
            for (int s = 0; s < 4; s++) {         // past the last piece: the last one again, not added
                const int64_t at = (int64_t)x.slot(min(s0 + s, x.parts - 1)) * kFewRows + row;
                ml[s] = __ldcg(a.part_ml + at);
#pragma unroll
                for (int i = 0; i < CK; i++) v[s][i] = __ldcg((const float4*)(a.part_o + at * D + min(c0 + 4 * per_row * i, D - 4)));
            }
            float top = M;
#pragma unroll
            for (int s = 0; s < 4; s++) top = fmaxf(top, ml[s].x);
            const float keep = weight(make_float2(M, 0.0f), top);
            L *= keep;
#pragma unroll
            for (int i = 0; i < CK; i++) { y[i].x *= keep; y[i].y *= keep; y[i].z *= keep; y[i].w *= keep; }
            M = top;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                if (s0 + s >= x.parts) continue;      // (a weight of zero counts: zero times a NaN)
                const float w = weight(ml[s], M);
                L += ml[s].y * w;
#pragma unroll
                for (int i = 0; i < CK; i++) {
                    y[i].x += v[s][i].x * w; y[i].y += v[s][i].y * w; y[i].z += v[s][i].z * w; y[i].w += v[s][i].w * w;
                }
            }
        }
        const float by = L == 0.0f ? 0.0f : 1.0f / L;
        T* out = (T*)(a.out + (int64_t)(x.r.begin + tok) * a.out_token + (int64_t)h * a.out_head);
#pragma unroll
        for (int i = 0; i < CK; i++)
            if (c0 + 4 * per_row * i < D)
                *(uint2*)(out + c0 + 4 * per_row * i) = make_uint2(pack2<T>(y[i].x * by, y[i].y * by), pack2<T>(y[i].z * by, y[i].w * by));
    }
}

template <int D, class T>
__global__ void __launch_bounds__(kFewThreads, few_blocks(D)) attend_few_kernel(AttendCall a) {
    extern __shared__ __align__(1024) uint8_t sm[];
    constexpr int KW = Few<D>::keys, KT = Few<D>::tile;
    __shared__ float s_m[kFewWarps][16], s_l[kFewWarps][16];
    __shared__ int s_bad[16], s_last;
    __shared__ Place s_place[kFewWarps][Few<D>::keys];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint8_t* ring_p = sm + warp * kFewStages * Few<D>::stage;
    const uint32_t ring = pf_smem(ring_p), qs = pf_smem(sm + Few<D>::ring);
    pdl_enter();
    const Share share = find_share<KT, kFewRows, kFewExtra, kFewThreads>(a, kFewLeast, (int64_t*)(sm + Few<D>::fixed));
    const int g = lane >> 2, quad = lane & 3;
    constexpr int CH = D / 8, RPI = 32 / CH;      // 16-byte pieces of a row, rows of a warp's copy

    Walk<KT, kFewRows, kFewExtra, kFewExtra> walk(a, share);
    for (Piece x; walk.next(x);) {
        __syncthreads();                          // the piece before is done with the rings and the rows
        const int32_t* table = a.table + (int64_t)x.b * a.table_stride;
        // the rows: past the tile's, zeros
        for (int i = tid; i < 16 * CH; i += kFewThreads) {
            const int r = i / CH, c = i % CH, R = x.row0 + r, tok = (int)a.group.div(R), h = x.head * (int)a.group.d + R - tok * (int)a.group.d;
            const bool there = r < x.rows;
            cp16(qs + few_at<D>(r, c), there ? a.q + (int64_t)(x.r.begin + tok) * a.q_token + (int64_t)h * a.q_head + c * 16 : a.q, there);
        }
        cp_commit();
        const int n = x.n, p_first = x.r.past + (int)a.group.div(x.row0), p_top = x.r.past + (int)a.group.div(x.row0 + x.rows - 1);
        const uint8_t *k_base = a.k.data + x.head * a.k.head, *v_base = a.v.data + x.head * a.v.head;
        // lane r: where key r of the warp's stage i lies, or -1; keys that no row sees are not fetched
        auto find = [&](int i) {
            const int j = x.tiles.tile(x.i0 + i) * KT + warp * KW + (lane & (KW - 1));
            int at = 0;
            const int page = i < n && seen(a, p_first, p_top, j) ? page_of(a, table, j, at) : -1;
            return page >= 0 ? Place{page * a.k.page + at * a.k.token, page * a.v.page + at * a.v.token} : Place{-1, -1};
        };
        // the places of the first stages are asked for together: one trip to the table
        Place ahead[kFewStages];
#pragma unroll
        for (int i = 0; i < kFewStages; i++) ahead[i] = find(i);
        // D 256: a row's fragments take as many registers as half of o: read again at each use
        constexpr bool HOLD = D <= 128;
        uint32_t qf[HOLD ? D / 16 : 1][4];
        int p[2];
#pragma unroll
        for (int i = 0; i < 2; i++) p[i] = g + 8 * i < x.rows ? x.r.past + (int)a.group.div(x.row0 + g + 8 * i) : -1;
        float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        uint32_t there = 0, there1 = 0;           // which of a stage's keys there are: of this stage, the next
        uint32_t into = ring, from = ring;        // the slot that is filled, the slot that is worked on
        auto on = [&](uint32_t slot) { return slot == ring + (kFewStages - 1) * Few<D>::stage ? ring : slot + Few<D>::stage; };
        // Two stages ahead, in one loop and with little unrolled: of a short call the larger part of the time
        // is the fetch of instructions that run once (one token at 1000, heads of 256: 15.8 us with the loop
        // unrolled by stages, stalled on instructions three times as long as they took to issue).
#pragma unroll 1
        for (int i = 1 - kFewStages; i < n; i++) {
            const uint32_t there2 = __ballot_sync(0xffffffffu, ahead[0].k >= 0);   // twice the same 16
            if (i + kFewStages - 1 < n) {
                __syncwarp();
                if (lane < KW) s_place[warp][lane] = ahead[0];
                __syncwarp();
                constexpr int ROUND = KW / RPI < 8 ? KW / RPI : 8;      // places that are loaded before they are used
#pragma unroll 1
                for (int e0 = 0; e0 < KW / RPI; e0 += ROUND) {
                    Place pl[ROUND];
#pragma unroll
                    for (int e = 0; e < ROUND; e++) pl[e] = s_place[warp][(e0 + e) * RPI + lane / CH];
#pragma unroll
                    for (int e = 0; e < ROUND; e++) {
                        const int r = (e0 + e) * RPI + lane / CH, c = lane % CH;
                        const bool is = pl[e].k >= 0;
                        cp16(into + few_at<D>(r, c), k_base + (is ? pl[e].k : 0) + c * 16, is);
                        cp16(into + Few<D>::half + few_at<D>(r, c), v_base + (is ? pl[e].v : 0) + c * 16, is);
                    }
                }
            }
            cp_commit();
            into = on(into);
#pragma unroll
            for (int e = 0; e + 1 < kFewStages; e++) ahead[e] = ahead[e + 1];
            ahead[kFewStages - 1] = find(i + 2 * kFewStages - 1);
            if (i >= 0) {
                cp_wait<kFewStages - 1>();
                if (i == 0) {
                    __syncthreads();              // the rows, which all warps brought
                    if (HOLD)
#pragma unroll
                        for (int k = 0; k < D / 16; k++) ldm4(qs + few_at<D>(lane & 15, 2 * k + (lane >> 4)), qf[k % (HOLD ? D / 16 : 1)]);
                }
                __syncwarp();
                const uint32_t ks = from, vs = ks + Few<D>::half;
                // (two sums of every other 16 values each: half the chain of products that wait for one another)
                float s[KW / 8][4] = {}, s_odd[KW / 8][4] = {};
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    uint32_t again[4];
                    if (!HOLD) ldm4(qs + few_at<D>(lane & 15, 2 * k + (lane >> 4)), again);
                    const uint32_t(&qk)[4] = HOLD ? qf[HOLD ? k : 0] : again;
#pragma unroll
                    for (int t = 0; t < KW / 16; t++) {
                        uint32_t b[4];
                        ldm4(ks + few_at<D>(16 * t + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)), b);
                        mma16<T>(k & 1 ? s_odd[2 * t] : s[2 * t], qk, b[0], b[1]);
                        mma16<T>(k & 1 ? s_odd[2 * t + 1] : s[2 * t + 1], qk, b[2], b[3]);
                    }
                }
                const int j0 = x.tiles.tile(x.i0 + i) * KT + warp * KW;
                // most stages lie where all rows see all keys: no comparison by key
                const bool all = there == 0xffffffffu && j0 + KW - 1 <= p_first &&
                                 (a.window <= 0 || p_top - j0 < a.window || j0 + KW <= a.sinks);
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int t = 0; t < KW / 8; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[t][e] = (s[t][e] + s_odd[t][e]) * a.scale_log2;
                if (!all)
#pragma unroll
                    for (int t = 0; t < KW / 8; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int r = t * 8 + quad * 2 + (e & 1);
                            if (!(there >> r & 1) || !sees(a, p[e >> 1], j0 + r)) s[t][e] = -INFINITY;
                        }
#pragma unroll
                for (int t = 0; t < KW / 8; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) top[e >> 1] = fmaxf(top[e >> 1], s[t][e]);
                float keep[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
                    const float mn = fmaxf(m[e], top[e]);
                    keep[e] = mn == -INFINITY ? 1.0f : exp2_of(m[e] - mn);
                    m[e] = mn;
                    top[e] = mn == -INFINITY ? 0.0f : mn - weight_lift<T>();
                    l[e] *= keep[e];
                }
#pragma unroll
                for (int t = 0; t < KW / 8; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        s[t][e] = exp2_of(s[t][e] - top[e >> 1]);
                        l[e >> 1] += s[t][e];
                    }
                // the weights, at most 2^lift, rounded to the cache's type for the second product (relative
                // error 2^-9 or 2^-12 each); l sums them unrounded
                uint32_t w[KW / 16][4];
#pragma unroll
                for (int t = 0; t < KW / 16; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) w[t][e] = pack2<T>(s[2 * t + (e >> 1)][2 * (e & 1)], s[2 * t + (e >> 1)][2 * (e & 1) + 1]);
#pragma unroll
                for (int c = 0; c < D / 8; c += 2) {
#pragma unroll
                    for (int e = 0; e < 4; e++) { o[c][e] *= keep[e >> 1]; o[c + 1][e] *= keep[e >> 1]; }
#pragma unroll
                    for (int t = 0; t < KW / 16; t++) {
                        uint32_t b[4];
                        ldm4t(vs + few_at<D>(16 * t + (lane & 7) + ((lane >> 3 & 1) << 3), c + (lane >> 4)), b);
                        mma16<T>(o[c], w[t], b[0], b[1]);
                        mma16<T>(o[c + 1], w[t], b[2], b[3]);
                    }
                }
                __syncwarp();
                from = on(from);
            }
            there = there1;
            there1 = there2;
        }
        cp_wait<0>();
        // the four warps' o, maxima and sums through shared memory: [16][D] f32 in the warp's own ring
        float* om = (float*)ring_p;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 2; e++) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
            if (quad == 0) { s_m[warp][g + 8 * e] = m[e] - weight_lift<T>(); s_l[warp][g + 8 * e] = l[e]; }
        }
#pragma unroll
        for (int c = 0; c < D / 8; c++)
#pragma unroll
            for (int e = 0; e < 2; e++) *(float2*)(om + (g + 8 * e) * Few<D>::part + 8 * c + 2 * quad) = make_float2(o[c][2 * e], o[c][2 * e + 1]);
        if (tid < 16) s_bad[tid] = 0;
        __syncthreads();
        // eight threads to a row, 4 values at a time
        const int row = tid >> 3, sub = tid & 7;
        float M = -INFINITY, f[kFewWarps], L = 0.0f;
        for (int w = 0; w < kFewWarps; w++) M = fmaxf(M, s_m[w][row]);
        for (int w = 0; w < kFewWarps; w++) {
            f[w] = s_m[w][row] == -INFINITY ? 0.0f : exp2_of(s_m[w][row] - M);
            L += s_l[w][row] * f[w];
        }
        float4 y[D / 32];
        bool fine = L - L == 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < kFewWarps; w++) {
                const float4 z = *(const float4*)(sm + w * kFewStages * Few<D>::stage + (row * Few<D>::part + sub * 4 + 32 * i) * 4);
                v.x += z.x * f[w]; v.y += z.y * f[w]; v.z += z.z * f[w]; v.w += z.w * f[w];
            }
            y[i] = v;
            const float z = (v.x - v.x) + (v.y - v.y) + (v.z - v.z) + (v.w - v.w);
            fine = fine && z == 0.0f;
        }
        if (!fine && row < x.rows) s_bad[row] = 1;
        if (__syncthreads_or(!fine && row < x.rows)) {
            for (int r = warp; r < x.rows; r += kFewWarps) {
                if (!s_bad[r]) continue;
                if (!met_hidden<D, T>(a, x, r, KT)) {      // it stays as it is
                    __syncwarp();
                    if (lane == 0) s_bad[r] = 0;
                    continue;
                }
                float c[D / 32], cm, cl;
                careful_row<D, T>(a, x, r, KT, c, cm, cl);
                for (int e = 0; e < D / 32; e++) ((float*)sm)[r * D + lane + 32 * e] = c[e];
                if (lane == 0) { s_m[0][r] = cm; s_l[0][r] = cl; }
            }
            __syncthreads();
            if (s_bad[row]) {
                M = s_m[0][row];
                L = s_l[0][row];
                for (int i = 0; i < D / 32; i++) y[i] = *(const float4*)(sm + (row * D + sub * 4 + 32 * i) * 4);
            }
        }
        if (x.parts > 1) {
            const int mine = x.slot(x.part);
            float* po = a.part_o + ((int64_t)mine * kFewRows + row) * D + sub * 4;
            for (int i = 0; i < D / 32; i++) __stcg((float4*)(po + 32 * i), y[i]);
            if (sub == 0) __stcg(a.part_ml + (int64_t)mine * kFewRows + row, make_float2(M, L));
            __syncthreads();
            if (tid == 0) {
                // releases what the block has written (it met at the barrier), acquires what the others have
                int before;
                asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(a.arrived + x.c0) : "memory");
                s_last = before == x.parts - 1;
                if (s_last) a.arrived[x.c0] = 0;
            }
            __syncthreads();
            if (!s_last) continue;
            join<D, T>(a, x);
            continue;
        }
        if (row < x.rows) {
            const int R = x.row0 + row, tok = (int)a.group.div(R), h = x.head * (int)a.group.d + R - tok * (int)a.group.d;
            T* out = (T*)(a.out + (int64_t)(x.r.begin + tok) * a.out_token + (int64_t)h * a.out_head) + sub * 4;
            const float by = L == 0.0f ? 0.0f : 1.0f / L;
            for (int i = 0; i < D / 32; i++)
                *(uint2*)(out + 32 * i) = make_uint2(pack2<T>(y[i].x * by, y[i].y * by), pack2<T>(y[i].z * by, y[i].w * by));
        }
    }
}

template <int D, class T> static cudaError_t few(const AttendCall& a, int sm_count, cudaStream_t stream) {
    const size_t smem = Few<D>::fixed + share_smem(a.n_seq, kFewThreads);
    static std::atomic<uint64_t> attr_set{0};
    if (cudaError_t e = ensure_dynamic_smem(attend_few_kernel<D, T>, (int)(Few<D>::fixed + share_smem(kCacheSeqs, kFewThreads)), attr_set)) return e;
    count_launch();
    return launch_with(pdl_mode() != 0, stream, attend_few_kernel<D, T>, dim3(sm_count * few_blocks(D)), dim3(kFewThreads), smem, a);
}
template <int D> static cudaError_t few_as(const AttendCall& a, int ggml_type, int sm_count, cudaStream_t stream) {
    return ggml_type == BIVMOE_F16 ? few<D, __half>(a, sm_count, stream) : few<D, __nv_bfloat16>(a, sm_count, stream);
}
cudaError_t launch_attend_few(const AttendCall& a, int head_dim, int ggml_type, int sm_count, cudaStream_t stream) {
    switch (head_dim) {
        case 64: return few_as<64>(a, ggml_type, sm_count, stream);
        case 128: return few_as<128>(a, ggml_type, sm_count, stream);
        default: return few_as<256>(a, ggml_type, sm_count, stream);
    }
}

}  // namespace bivmoe
