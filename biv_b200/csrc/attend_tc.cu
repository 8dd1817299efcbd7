// Attention over the pages for tiles of 128 and 256 rows on the fifth-generation tensor cores.
//
//   S = Q K^T (128 rows x 128 keys),  P = 2^(scale S - m),  O += P V,  o = O / sum P
//
// One block per SM takes its share of the work (cache.cuh) and has four kinds of warps:
//
//   warps 0-7    two groups of 128 threads, a thread to a row: S from tensor memory, its maximum, the
//                powers, P as 16-bit values back into tensor memory over S; at a piece's start the
//                rows' Q into shared memory, at its end O out.
//   warp 8       one lane issues the MMAs.  K and V stand in shared memory in rows of 64 values
//                (128-byte swizzle): K is read along the values (K-major), V along the keys (MN-major),
//                so that neither is turned; P is read from tensor memory.
//   warp 9       finds where a tile's keys lie, ahead of the copies.
//   warps 12-15  bring K and V from the pages, 128 keys x 64 values (16 KB) a slot, in a ring of eight: by
//                the copy engine, a box for each page's part, where pages are of 16 tokens and more and
//                the tile ends before the rows' last key; else cp.async in 16-byte pieces.
//
// Heads of up to 128 values: two tiles of 128 rows at once, a group each, so that one group's powers
// run while the other's products do.  Heads of 256 values, whose O alone takes half of tensor memory,
// and pieces of up to 128 rows: one tile with two S, the next product into one while the first group
// works on the other.
// Bound by neither pipe alone: with heads of 128 the tensor cores and the special-function unit (a power
// for each score, 1024 clocks a tile of 128 x 128) are each busy 40 % of the time, and S's way out of tensor
// memory and P's way in lengthen a tile's chain: 2048 tokens at 30000, 32 / 8 heads, 1.04 TFLOP, 1040 us
// (1210 to 1250 under the power cap), 0.61 of the measured bf16 peak.  With heads of 256 a key tile is
// 128 KB, longer on its way from L2 than in the products: a prompt of 4096, 16 / 2 heads, 182 us.
// m is not the running maximum itself but one that follows it when it has grown by more than 2^8:
// O is then scaled in tensor memory, which happens a few times at a piece's start and rarely after (P
// is lifted with room for that; its sum and O are held in f32).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <stddef.h>

#include "cache.cuh"
#include "common.cuh"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace bivmoe {

constexpr int AT_KEYS = 128, AT_SLOT = AT_KEYS * 128, AT_SLOTS = 8;
constexpr int AT_THREADS = 512, AT_MMA_WARP = 8, AT_PAGE_WARP = 9, AT_COPY_WARP = 12, AT_COPY_WARPS = 4;
constexpr int AT_ROW_REGS = 192, AT_OTHER_REGS = 64;
static_assert(AT_ROW_REGS * 256 + AT_OTHER_REGS * 256 <= 512 * 128, "setmaxnreg would wait for registers that nobody gives");
constexpr int AT_HEAD = 1024, AT_PAGES = 8;    // key tiles whose addresses stand ready
constexpr float AT_GROWTH = 8.0f;     // powers of two
enum { AT_SITE_COPY = 31, AT_SITE_MMA, AT_SITE_ROWS, AT_SITE_PAGES };

// Where a tile's keys and values lie: bytes from the head's first page on, -1 where there is none; or the
// boxes that the copy engine fetches, the pool's number of pages for one that is not there (it writes zeros).
struct AtPlaces {
    union {
        struct { int64_t k[AT_KEYS], v[AT_KEYS]; };
        struct { int page[16], row[16]; };
    };
};
template <int D> struct At {
    static constexpr int tiles = D == 256 ? 1 : 2;           // of 128 rows
    static constexpr int rows = 128 * tiles;
    static constexpr int chunks = D / 64;                    // slots of a tile of K, or of V
    // Key tiles that a tile costs besides.  us with 0 / 4 / 6 / 9: a prompt of 4096, heads of 256, 404 / 170 / 174 /
    // 207; with 0 / 2 / 4 / 6: ragged prompts, heads of 64, 79 / 60 / 62 / 66.
    static constexpr int extra = D == 256 ? 4 : 3;
    // Key tiles that are not worth a cut.  us with 4 or 3 / 6 or 5 / 9 or 8: 48 rows at 1000 in eight requests, heads of
    // 256, 38.1 / 27.6 / 27.6; a windowed prompt, heads of 128, 289 / 259 / 247; ragged prompts 60 / 62 / 69.
    static constexpr int snap = D == 256 ? 6 : 5;
    static constexpr int q_tile = 128 * D * 2;
    static constexpr int fixed = AT_HEAD + tiles * q_tile + AT_SLOTS * AT_SLOT + (int)sizeof(AtPlaces) * AT_PAGES;
};

// the pools for the copy engine: boxes of `rows` tokens x 64 values; rows 0: none
struct AtMaps {
    CUtensorMap k, v;
    int rows;
};
struct AtHead {
    uint64_t full[AT_SLOTS], empty[AT_SLOTS];
    // [0], [1]: of the two tiles of a pair; [2], [3]: of the two S of a single tile.  Apart, because the
    // second group passes single tiles by: a parity tells a phase from the next one only.
    uint64_t s_full[4], p_half[4], p_full[4], q_full[2], pv_done[2], drained;
    uint64_t page_full[AT_PAGES], page_empty[AT_PAGES];
    // Which keys of a tile lie in pages that there are, or are seen by no row; read 16 bytes at once.  The
    // addresses are at most eight tiles ahead of the copies, these at most five ahead of the rows.
    alignas(16) uint32_t there[16][4];
    int boxes[AT_PAGES];              // of a key tile that the copy engine fetches, or 0
    uint32_t tmem;
    int abort;
    int mending;                      // warps that make rows again, which may take as long as there are keys
};
static_assert(sizeof(AtHead) <= AT_HEAD && offsetof(AtHead, there) % 16 == 0, "");

// Each role's registers are dealt out in its own branch: where branches meet, the compiler reckons with
// the fewest.
__device__ __forceinline__ void at_fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AT_OTHER_REGS)); }
// Every role's waits look at the clock, once in 64 tries that found nothing: a role that ends early does not
// leave the others without one that gives up.  The clock stands while rows are made again: that is bounded
// by the keys they see, and could take longer than any other wait.  (A look is a call: written out at every
// wait it made a prompt of 4096, heads of 256, 188 us instead of 181.)
__device__ __noinline__ uint64_t at_look(const AtHead* h, uint32_t look, uint64_t t0) {   // where the clock began; 0: gives up
    WaitClock clock{t0};
    if (*(const volatile int*)&h->abort) return 0;
    return clock.late(look, pf_now_ns(), *(const volatile int*)&h->mending != 0) ? 0 : clock.t0;
}
template <bool SLEEP> struct AtWait {
    uint64_t* bar;
    uint32_t parity;
    const AtHead* h;
    uint64_t t0 = 0;
    __device__ __forceinline__ bool ready() const { return pf_bar_try(bar, parity); }
    __device__ __forceinline__ bool late(uint32_t look) { return !(t0 = at_look(h, look, t0)); }
    __device__ __forceinline__ void pause() const { if (SLEEP) __nanosleep(32); }
    __device__ __forceinline__ bool all(bool v) const { return __all_sync(0xffffffffu, v); }
};
__device__ __forceinline__ bool at_wait(uint64_t* bar, uint32_t parity, const AtHead* h) {
    return bounded_wait<64>(AtWait<false>{bar, parity, h});
}
template <bool SLEEP = false> __device__ __forceinline__ bool at_wait_warp(uint64_t* bar, uint32_t parity, const AtHead* h) {
    return bounded_wait_together<64>(AtWait<SLEEP>{bar, parity, h});
}
// One lane's arrival for its warp, which is together again after it: what follows may be an instruction that
// a whole warp has to execute at once (tcgen05.ld, .st), and a branch that one lane takes does not by
// itself end together.
__device__ __forceinline__ void at_arrive(uint64_t* bar) {
    if ((threadIdx.x & 31) == 0) pf_bar_arrive(bar);
    __syncwarp();
}
// the thread's arrival, once its copies so far have landed
__device__ __forceinline__ void at_cp_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(pf_smem(bar)) : "memory");
}
// 64 values of `rows` tokens of a page's head, zeros where there is no such page
__device__ __forceinline__ void at_box(uint32_t dst, const CUtensorMap* map, int value, int token, int head, int page, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
                     "r"(dst), "l"(map), "r"(value), "r"(token), "r"(head), "r"(page), "r"(pf_smem(bar)) : "memory");
}
// what threads have written to shared memory, or have seen written, before what the tensor cores read
__device__ __forceinline__ void at_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void at_tmem_st32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void at_tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// A in tensor memory
__device__ __forceinline__ void at_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc),
        "r"(accumulate)
        : "memory");
}
// kind::f16, f32 accumulator, A and B of T; B along its rows (MN-major) or along K
template <class T> __device__ __forceinline__ constexpr uint32_t at_idesc(int n, bool b_mn);
template <> __device__ __forceinline__ constexpr uint32_t at_idesc<__half>(int n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
template <> __device__ __forceinline__ constexpr uint32_t at_idesc<__nv_bfloat16>(int n, bool b_mn) {
    return at_idesc<__half>(n, b_mn) | (1u << 7) | (1u << 10);
}
// MN-major, 128-byte swizzle: 64 values of N are a row of 128 bytes, 8 keys a 1024-byte atom; 1024 bytes
// from 8 keys to the next 8, a slot from 64 values to the next 64.  A K step of 16 keys is 2048 bytes.
__device__ __forceinline__ uint64_t at_desc_v(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(AT_SLOT >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// 16-byte piece `c` of row `r` of 128 rows in tiles of 64 values, 128-byte swizzle
__device__ __forceinline__ uint32_t at_piece(uint32_t tile, int r, int c) {
    return tile + (c >> 3) * (128 * 128) + r * 128 + (((c ^ r) & 7) << 4);
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// place q of the 2 n tiles of K and V in the order the products take them
struct AtTurn { bool v; int j; };
__device__ __forceinline__ AtTurn at_turn(int q, int n, bool pair) {
    if (pair) return AtTurn{(q & 1) != 0, q >> 1};
    if (q == 0) return AtTurn{false, 0};
    if (q == 2 * n - 1) return AtTurn{true, n - 1};
    return q & 1 ? AtTurn{false, (q + 1) >> 1} : AtTurn{true, (q >> 1) - 1};
}

template <int D, class T>
__global__ void __launch_bounds__(AT_THREADS, 1) attend_tc_kernel(const __grid_constant__ AttendCall a, const __grid_constant__ AtMaps maps) {
    extern __shared__ __align__(1024) uint8_t sm[];
    AtHead& H = *(AtHead*)sm;
    constexpr int NT = At<D>::tiles, TR = At<D>::rows, CH = At<D>::chunks;
    uint8_t* q_sm = sm + AT_HEAD;
    uint8_t* ring = q_sm + NT * At<D>::q_tile;
    AtPlaces* places = (AtPlaces*)(ring + AT_SLOTS * AT_SLOT);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_enter();
    // the share is looked at once a piece: it stands in shared memory, the rows' registers are full
    __shared__ Share share;
    {
        const Share found = find_share<AT_KEYS, TR, At<D>::extra, AT_THREADS>(a, 1, (int64_t*)(sm + At<D>::fixed));
        if (found.lo >= found.hi) return;
        if (tid == 0) share = found;
    }
    if (tid == 0) {
        for (int i = 0; i < AT_SLOTS; i++) { pf_bar_init(&H.full[i], 32); pf_bar_init(&H.empty[i], 1); }
        for (int i = 0; i < 2; i++) {
            pf_bar_init(&H.q_full[i], 4);
            pf_bar_init(&H.pv_done[i], 1);
        }
        for (int i = 0; i < 4; i++) { pf_bar_init(&H.s_full[i], 1); pf_bar_init(&H.p_half[i], 4); pf_bar_init(&H.p_full[i], 4); }
        for (int i = 0; i < AT_PAGES; i++) { pf_bar_init(&H.page_full[i], 1); pf_bar_init(&H.page_empty[i], 2 * CH); }
        pf_bar_init(&H.drained, 1);
        H.abort = H.mending = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == AT_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pf_smem(&H.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pf_fence_before();
    __syncthreads();
    pf_fence_after();
    const uint32_t tmem = H.tmem;
    auto give_up = [&](int site) {
        if (lane == 0) {
            atomicExch(a.status, site);
            *(volatile int*)&H.abort = 1;
        }
    };
    Walk<AT_KEYS, TR, At<D>::extra, At<D>::snap> walk(a, share);

    if (warp == AT_PAGE_WARP) {
        at_fewer_regs();
        // ---- addresses: four keys a lane, once for K and V and all their slots
        uint32_t ktile = 0;                       // key tiles of the pieces before
        bool ok = true;
        for (Piece x; ok && walk.next(x);) {
            const int n = max(x.n, 0), p_top = x.r.past + (int)a.group.div(x.row0 + x.rows - 1);
            const int32_t* table = a.table + (int64_t)x.b * a.table_stride;
            for (int j = 0; j < n; j++, ktile++) {
                const int e = ktile % AT_PAGES, key0 = x.tiles.tile(x.i0 + j) * AT_KEYS;
                // The copy engine fetches tiles that end before the rows' last key: what lies behind that one in
                // its page belongs to nobody, may be anything, and has to be zeros here.
                const bool boxes = maps.rows && key0 + AT_KEYS - 1 <= p_top;
                int page[4], at[4];
                uint32_t known[4];
                if (boxes) {
                    const int n_box = AT_KEYS / maps.rows;
                    page[0] = lane < n_box ? page_of(a, table, key0 + lane * maps.rows, at[0]) : -1;
                    const uint32_t there = __ballot_sync(0xffffffffu, page[0] >= 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) known[i] = __ballot_sync(0xffffffffu, there >> ((32 * i + lane) / maps.rows) & 1);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int key = key0 + 32 * i + lane;
                        page[i] = key <= p_top ? page_of(a, table, key, at[i]) : -1;
                        known[i] = __ballot_sync(0xffffffffu, page[i] >= 0 || key > p_top);
                    }
                }
                if (!at_wait_warp<true>(&H.page_empty[e], ((ktile / AT_PAGES) & 1) ^ 1, &H)) {
                    give_up(AT_SITE_PAGES);
                    ok = false;
                    break;
                }
                if (boxes) {
                    if (lane < 16) { places[e].page[lane] = page[0] >= 0 ? page[0] : (int)a.k.n_pages; places[e].row[lane] = at[0]; }
                } else
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    places[e].k[32 * i + lane] = page[i] >= 0 ? page[i] * a.k.page + at[i] * a.k.token : -1;
                    places[e].v[32 * i + lane] = page[i] >= 0 ? page[i] * a.v.page + at[i] * a.v.token : -1;
                }
                if (lane == 0) H.boxes[e] = boxes ? AT_KEYS / maps.rows : 0;
                if (lane == 0) *(uint4*)H.there[ktile & 15] = make_uint4(known[0], known[1], known[2], known[3]);
                __syncwarp();
                at_arrive(&H.page_full[e]);
            }
        }
    } else if (warp >= AT_COPY_WARP) {
        at_fewer_regs();
        // ---- copies
        uint32_t base = 0, ktile = 0;             // slots, key tiles of the pieces before
        uint32_t last = 0, fills = 0;             // the last slot this warp filled, how many
        bool ok = true;
        for (Piece x; ok && walk.next(x);) {
            const int n = max(x.n, 0), total = 2 * n * CH;
            const bool pair = NT == 2 && x.rows > 128;
            // this warp's slots: every fourth of the block's
            for (int i = (int)((warp - AT_COPY_WARP - base) & 3); i < total; i += AT_COPY_WARPS) {
                const uint32_t gs = base + i, slot = gs % AT_SLOTS;
                const AtTurn turn = at_turn(i / CH, n, pair);
                const int c = i % CH;
                const uint32_t kt = ktile + turn.j;
                if (!at_wait_warp<true>(&H.page_full[kt % AT_PAGES], (kt / AT_PAGES) & 1, &H) ||
                    !at_wait_warp<true>(&H.empty[slot], ((gs / AT_SLOTS) & 1) ^ 1, &H)) {
                    give_up(AT_SITE_COPY);
                    ok = false;
                    break;
                }
                last = gs;
                fills++;
                const AtPlaces& pl = places[kt % AT_PAGES];
                if (const int n_box = H.boxes[kt % AT_PAGES]) {
                    if (lane == 0) pf_bar_expect_tx(&H.full[slot], AT_SLOT);
                    __syncwarp();
                    if (lane < n_box)
                        at_box(pf_smem(ring + slot * AT_SLOT) + lane * maps.rows * 128, turn.v ? &maps.v : &maps.k, c * 64, pl.row[lane],
                               x.head, pl.page[lane], &H.full[slot]);
                    if (lane) pf_bar_arrive(&H.full[slot]);
                    __syncwarp();
                    at_arrive(&H.page_empty[kt % AT_PAGES]);
                    continue;
                }
                const int64_t* place = turn.v ? pl.v : pl.k;
                const uint8_t* from = (turn.v ? a.v.data + x.head * a.v.head : a.k.data + x.head * a.k.head) + c * 128 + ((lane & 7) << 4);
                const uint32_t dst = pf_smem(ring + slot * AT_SLOT) + ((lane & 7) << 4);
                // lanes 8 g to 8 g + 7: the eight pieces of a row; eight addresses at a time, so that their loads'
                // latency passes once for eight copies
#pragma unroll
                for (int s0 = 0; s0 < AT_KEYS / 4; s0 += 8) {
                    int64_t o[8];
#pragma unroll
                    for (int s = 0; s < 8; s++) o[s] = place[4 * (s0 + s) + (lane >> 3)];
#pragma unroll
                    for (int s = 0; s < 8; s++) {
                        const int r = 4 * (s0 + s) + (lane >> 3);
                        cp16((dst + r * 128) ^ ((r & 7) << 4), from + max(o[s], (int64_t)0), o[s] >= 0);
                    }
                }
                at_cp_arrive(&H.full[slot]);
                __syncwarp();
                at_arrive(&H.page_empty[kt % AT_PAGES]);
            }
            base += total;
            ktile += n;
        }
        // Nothing is in flight when the block ends, whatever ended the loops: nobody may have waited for the last slots.
        asm volatile("cp.async.wait_all;" ::: "memory");
        wait_for_last_fills<AT_SLOTS, AT_COPY_WARPS>(last, fills, [&](uint32_t slot, uint32_t parity) { pf_bar_wait(&H.full[slot], parity); });
        __syncwarp();
    } else if (warp == AT_MMA_WARP) {
        at_fewer_regs();
        // ---- products
        uint32_t base = 0, pieces[2] = {0, 0};    // slots, Q tiles of the pieces before
        uint32_t used[3] = {0, 0, 0};             // S: of each tile of the pairs; the two of single tiles
        const uint32_t o_at = tmem, s_at = tmem + 256;
        bool ok = true;
        for (Piece x; ok && walk.next(x);) {
            const int n = max(x.n, 0);
            if (!n) continue;
            const bool pair = NT == 2 && x.rows > 128;
            if (pf_elect()) {
                uint32_t cp[4] = {used[0], used[0], used[1], used[2]};
                auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = ok && at_wait(bar, parity, &H); };
                auto slot_of = [&](int q, int c) { return (base + q * CH + c) % AT_SLOTS; };
                // a tile of K or V, all its slots
                auto landed = [&](int q) {
                    for (int c = 0; c < CH; c++) {
                        const uint32_t gs = base + q * CH + c;
                        wait(&H.full[gs % AT_SLOTS], (gs / AT_SLOTS) & 1);
                    }
                    at_fence_async();
                };
                auto free = [&](int q) {
                    for (int c = 0; c < CH; c++) pf_commit(&H.empty[slot_of(q, c)]);
                };
                // `s`: the S by its barriers (AtHead); the odd ones stand 128 columns on
                auto scores = [&](int q, int t, int s) {          // S_s = Q_t K^T
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        const uint32_t qa = pf_smem(q_sm + t * At<D>::q_tile + c * (128 * 128)), ka = pf_smem(ring + slot_of(q, c) * AT_SLOT);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            pf_mma_bf16(s_at + (s & 1) * 128, pf_desc_sw128(qa + 32 * k), pf_desc_sw128(ka + 32 * k), at_idesc<T>(AT_KEYS, false),
                                        c || k);
                    }
                    pf_commit(&H.s_full[s]);
                };
                // O_t += P_s V: the first 64 keys' weights are there before the others are made
                auto values = [&](int q, int t, int s, bool first) {
                    const uint32_t va = pf_smem(ring + slot_of(q, 0) * AT_SLOT), parity = cp[s]++ & 1;
                    if (t == 0) landed(q);                // (the second tile's turn: it has)
                    wait(&H.p_half[s], parity);
                    pf_fence_after();
                    if (!ok) return;
#pragma unroll
                    for (int k = 0; k < AT_KEYS / 16; k++) {
                        if (k == AT_KEYS / 32) {
                            wait(&H.p_full[s], parity);
                            pf_fence_after();
                            if (!ok) return;
                        }
                        at_mma_ts(o_at + t * D, s_at + (s & 1) * 128 + 8 * k, at_desc_v(va + 2048 * k), at_idesc<T>(D, true), !first || k);
                    }
                    pf_commit(&H.pv_done[t]);
                };
                wait(&H.q_full[0], pieces[0] & 1);
                if (pair) wait(&H.q_full[1], pieces[1] & 1);
                at_fence_async();
                if (pair) {
                    landed(0);
                    if (ok) { scores(0, 0, 0); scores(0, 1, 1); free(0); }
                    for (int j = 0; j < n && ok; j++) {
                        const bool more = j + 1 < n;
                        for (int t = 0; t < 2 && ok; t++) {
                            values(2 * j + 1, t, t, j == 0);
                            if (!ok) break;
                            if (t == 1) free(2 * j + 1);
                            if (more) {
                                if (t == 0) landed(2 * j + 2);
                                if (!ok) break;
                                scores(2 * j + 2, t, t);
                                if (t == 1) free(2 * j + 2);
                            }
                        }
                    }
                } else {
                    landed(0);
                    if (ok) { scores(0, 0, 2); free(0); }
                    for (int j = 0; j < n && ok; j++) {
                        const int kq = 2 * j + 1, vq = j + 1 < n ? 2 * j + 2 : 2 * n - 1;
                        if (j + 1 < n) {
                            landed(kq);
                            if (!ok) break;
                            scores(kq, 0, 2 + ((j + 1) & 1));
                            free(kq);
                        }
                        values(vq, 0, 2 + (j & 1), j == 0);
                        if (ok) free(vq);
                    }
                }
                if (!ok) {
                    atomicExch(a.status, AT_SITE_MMA);
                    *(volatile int*)&H.abort = 1;
                }
            }
            __syncwarp();
            base += 2 * n * CH;
            pieces[0]++;
            pieces[1] += pair;
            if (pair) used[0] += n;
            else { used[1] += (n + 1) / 2; used[2] += n / 2; }
            ok = pf_together(!*(volatile int*)&H.abort);
        }
        // nothing is in flight when the block ends, whatever ended its loops
        if (pf_elect()) pf_commit(&H.drained);
        __syncwarp();
        pf_bar_wait(&H.drained, 0);
        __syncwarp();
    } else if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AT_ROW_REGS));
        // ---- rows
        const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        uint32_t cs[3] = {0, 0, 0}, cpv = 0, ktile = 0;   // S of the pairs' tile, the two of single tiles
        const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);       // a masked score times it is no NaN
        bool ok = true;
        for (Piece x; ok && walk.next(x);) {
            const int n = max(x.n, 0);
            const bool pair = NT == 2 && x.rows > 128;
            const int t = pair ? wg : 0;
            if (wg && !pair) {                        // the other group's piece alone
                ktile += n;
                continue;
            }
            const int R = x.row0 + t * 128 + row, last = x.row0 + x.rows - 1;
            const bool mine = R <= last, any = x.row0 + t * 128 + (warp & 3) * 32 <= last;
            const int Rc = min(R, last), tok = (int)a.group.div(Rc), h = x.head * (int)a.group.d + Rc - tok * (int)a.group.d;
            const int p = x.r.past + tok;
            const int p_first = x.r.past + (int)a.group.div(min(x.row0 + t * 128, last)),
                      p_top = x.r.past + (int)a.group.div(min(x.row0 + t * 128 + 127, last));
            float m = -INFINITY, l = 0.0f;
            constexpr float lift = weight_lift<T>() - AT_GROWTH;  // so high with the growth
            const uint32_t qs = pf_smem(q_sm + t * At<D>::q_tile);
            constexpr int PR = D / 8, RPI = 32 / PR;              // pieces of a row, rows of a warp's access
            if (n) {
                // Q: the warp's own 32 rows; past the tile's, zeros
#pragma unroll 8
                for (int i = 0; i < 32 / RPI; i++) {
                    const int r = (warp & 3) * 32 + i * RPI + lane / PR, Q = min(x.row0 + t * 128 + r, last), qt = (int)a.group.div(Q);
                    cp16(at_piece(qs, r, lane % PR),
                            a.q + (int64_t)(x.r.begin + qt) * a.q_token + (int64_t)(x.head * (int)a.group.d + Q - qt * (int)a.group.d) * a.q_head +
                                (lane % PR) * 16, x.row0 + t * 128 + r <= last);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                if (a.scale_log2 < 0.0f)              // of a negative scale the sign goes to the rows
#pragma unroll 1
                    for (int i = 0; i < 32 / RPI; i++) {
                        const uint32_t at = at_piece(qs, (warp & 3) * 32 + i * RPI + lane / PR, lane % PR);
                        const uint4 w = lds128(at);   // (the lane's own copy)
                        sts128(at, make_uint4(w.x ^ 0x80008000u, w.y ^ 0x80008000u, w.z ^ 0x80008000u, w.w ^ 0x80008000u));
                    }
                at_fence_async();
                __syncwarp();
                at_arrive(&H.q_full[t]);
            }
            for (int j = 0; j < n; j++) {
                const int s = pair ? t : 2 + (j & 1);
                uint32_t& count = pair ? cs[0] : j & 1 ? cs[2] : cs[1];
                if (!at_wait_warp(&H.s_full[s], count & 1, &H)) { ok = false; break; }
                count++;
                // Every product's end is waited for, and before the next one can begin: a parity tells a phase
                // from the one before or after it only.  (Pairs: the scores follow it.  Single tiles: it is
                // followed by the next scores, so that the tensor cores do not wait for this.)
                auto before = [&] { return !j || pair || at_wait_warp(&H.pv_done[t], (cpv + j - 1) & 1, &H); };
                if (any) {
                    pf_fence_after();
                    const uint32_t s_at = tmem + 256 + (s & 1) * 128 + lanes;
                    int v[128];
#pragma unroll
                    for (int e = 0; e < 4; e++) pf_tmem_ld32(s_at + 32 * e, *(int(*)[32])(v + 32 * e));
                    // (looked at while S is on its way)
                    const int key0 = x.tiles.tile(x.i0 + j) * AT_KEYS;
                    const uint4 there = *(const uint4*)H.there[(ktile + j) & 15];
                    const bool all = (there.x & there.y & there.z & there.w) == 0xffffffffu && key0 + AT_KEYS - 1 <= p_first &&
                                     (a.window <= 0 || p_top - key0 < a.window || key0 + AT_KEYS <= a.sinks);
                    pf_tmem_wait_ld();
                    if (!all) {
                        const uint32_t tw[4] = {there.x, there.y, there.z, there.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int k0 = key0 + 32 * e;
                            uint32_t see = bits_below(p + 1 - k0) & tw[e];
                            if (a.window > 0) see &= ~bits_below(p - a.window + 1 - k0) | bits_below(a.sinks - k0);
#pragma unroll
                            for (int i = 0; i < 32; i++) v[32 * e + i] = see >> i & 1 ? v[32 * e + i] : (int)0xff800000u;   // -infinity
                        }
                    }
                    float top[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 128; i += 2) top[i / 2 & 3] = max3(top[i / 2 & 3], __int_as_float(v[i]), __int_as_float(v[i + 1]));
                    const float grown = fmaxf(max3(top[0], top[1], top[2]), top[3]);
                    if (j == 0) m = grown;
                    const bool far = (grown - m) * scale > AT_GROWTH;
                    if (__any_sync(0xffffffffu, far)) {
                        // O follows, once the product before has been added
                        if (!before()) { ok = false; break; }
                        pf_fence_after();
                        const float by = far ? (m == -INFINITY ? 0.0f : exp2_of((m - grown) * scale)) : 1.0f;
                        if (far) m = grown;
                        l *= by;
                        const uint32_t o_at = tmem + t * D + lanes;
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            int o[32];
                            pf_tmem_ld32(o_at + c, o);
                            pf_tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = __float_as_int(__int_as_float(o[i]) * by);
                            at_tmem_st32(o_at + c, (const uint32_t*)o);
                        }
                        at_tmem_wait_st();
                    }
                    const float minus = m == -INFINITY ? 0.0f : lift - m * scale;
                    const f32x2 sc = pk(scale, scale), mi = pk(minus, minus);
                    f32x2 sum[2] = {0, 0};
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        uint32_t w[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            const f32x2 z = fma2(pk(__int_as_float(v[64 * e + 2 * i]), __int_as_float(v[64 * e + 2 * i + 1])), sc, mi);
                            const f32x2 y = pk(exp2_of(lo_of(z)), exp2_of(hi_of(z)));
                            sum[i & 1] = add2(sum[i & 1], y);
                            // the weights rounded to the cache's type for the second product (relative error
                            // 2^-9 or 2^-12 each); l sums them unrounded
                            w[i] = pack2<T>(lo_of(y), hi_of(y));
                        }
                        at_tmem_st32(s_at + 32 * e, w);
                        if (e == 0) {
                            at_tmem_wait_st();
                            if (!before()) { ok = false; break; }
                            pf_fence_before();
                            at_arrive(&H.p_half[s]);
                        }
                    }
                    if (!ok) break;
                    sum[0] = add2(sum[0], sum[1]);
                    l += lo_of(sum[0]) + hi_of(sum[0]);
                    at_tmem_wait_st();
                } else {
                    if (!before()) { ok = false; break; }
                    __syncwarp();
                    at_arrive(&H.p_half[s]);
                }
                pf_fence_before();
                __syncwarp();
                at_arrive(&H.p_full[s]);
            }
            if (!ok) { give_up(AT_SITE_ROWS); break; }
            ktile += n;
            if (n) {
                if (!at_wait_warp(&H.pv_done[t], (cpv + n - 1) & 1, &H)) { give_up(AT_SITE_ROWS); ok = false; break; }
                cpv += n;
                pf_fence_after();
            }
            if (!any) continue;
            // ---- O out, through the shared memory of the warp's rows of Q, so that rows are written whole
            const bool cut = x.parts > 1;
            const float by = cut ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t out_at = (int64_t)(x.r.begin + tok) * a.out_token + (int64_t)h * a.out_head;
            const int r0 = t * 128 + (warp & 3) * 32, rows = min(32, x.rows - r0);     // the warp's, of the tile
            const int64_t place0 = (int64_t)x.slot(x.part) * TR + r0;
            float odd = l * 0.0f;                     // NaN as soon as something is not finite
            __syncwarp();
            // unfinished sums go out in f32, in two halves of the row, results in one
#pragma unroll 1
            for (int half = 0; half < (cut ? 2 : 1); half++) {
                const int c0 = half * (D / 2), c1 = cut ? c0 + D / 2 : D;
                // (32 columns to a trip to tensor memory; with 64 and 128 the loop, which runs once a piece, has more
                // instructions to fetch: ragged prompts 61.5 -> 69.3 us)
                constexpr int WIDE = 32;
#pragma unroll 1
                for (int c = c0; c < c1; c += WIDE) {
                    int o[WIDE];
                    if (n) {
#pragma unroll
                        for (int i = 0; i < WIDE; i += 32) pf_tmem_ld32(tmem + t * D + lanes + c + i, *(int(*)[32])(o + i));
                        pf_tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < WIDE; i++) o[i] = 0;
                    }
                    float bad[4] = {};
#pragma unroll
                    for (int i = 0; i < WIDE; i++) bad[i & 3] = fmaf(__int_as_float(o[i]), 0.0f, bad[i & 3]);
                    odd += (bad[0] + bad[1]) + (bad[2] + bad[3]);
                    if (cut) {
#pragma unroll
                        for (int i = 0; i < WIDE / 4; i++)
                            sts128(at_piece(qs, row, (c - c0) / 4 + i), make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
                    } else {
                        auto two = [&](int i) { return pack2<T>(__int_as_float(o[i]) * by, __int_as_float(o[i + 1]) * by); };
#pragma unroll
                        for (int i = 0; i < WIDE / 8; i++)
                            sts128(at_piece(qs, row, c / 8 + i), make_uint4(two(8 * i), two(8 * i + 2), two(8 * i + 4), two(8 * i + 6)));
                    }
                }
                // (a row that may be made again below is not written here: `out` may be where its q stands)
                const uint32_t again = cut ? 0u : __ballot_sync(0xffffffffu, odd != 0.0f);
                __syncwarp();
#pragma unroll 1
                for (int i0 = 0; i0 < 32 / RPI; i0 += 8) {
                    uint4 w[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i] = lds128(at_piece(qs, (warp & 3) * 32 + (i0 + i) * RPI + lane / PR, lane % PR));
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int r = (i0 + i) * RPI + lane / PR, c = lane % PR;
                        const int64_t to = __shfl_sync(0xffffffffu, out_at, r);
                        if (r < rows && !(again >> r & 1)) {
                            if (cut) __stcg((uint4*)(a.part_o + (place0 + r) * D + c0 + 4 * c), w[i]);
                            else *(uint4*)(a.out + to + 16 * c) = w[i];
                        }
                    }
                }
                __syncwarp();
            }
            if (cut && mine) __stcg(a.part_ml + place0 + lane, make_float2(m * scale - lift, l));
            const uint32_t odd_rows = __ballot_sync(0xffffffffu, mine && odd != 0.0f);
            if (odd_rows && lane == 0) atomicAdd(&H.mending, 1);
            for (uint32_t bad = odd_rows; bad; bad &= bad - 1) {
                __syncwarp();
                const int of = __ffs(bad) - 1, r = r0 + of;
                const int64_t out_of = __shfl_sync(0xffffffffu, out_at, of), at = place0 + of;
                if (!met_hidden<D, T>(a, x, r, AT_KEYS)) {            // it stays as it is, and still stands in shared memory
                    if (!cut && lane < PR) *(uint4*)(a.out + out_of + 16 * lane) = lds128(at_piece(qs, (warp & 3) * 32 + of, lane));
                    continue;
                }
                float o[D / 32], cm, cl;
                careful_row<D, T>(a, x, r, AT_KEYS, o, cm, cl);
                const float inv = cl == 0.0f ? 0.0f : 1.0f / cl;
                for (int e = 0; e < D / 32; e++) {
                    if (cut) __stcg(a.part_o + at * D + lane + 32 * e, o[e]);
                    else ((T*)(a.out + out_of))[lane + 32 * e] = from_f32<T>(o[e] * inv);
                }
                if (cut && lane == 0) __stcg(a.part_ml + at, make_float2(cm, cl));
            }
            if (odd_rows && lane == 0) atomicAdd(&H.mending, -1);
            if (!cut) continue;
            // the warp that is last with these 32 rows joins their pieces, in the pieces' order
            __threadfence();
            __syncwarp();
            int last_one = 0;
            int32_t* arrived = a.arrived + x.c0 * 8 + t * 4 + (warp & 3);
            if (lane == 0) {
                last_one = atomicAdd(arrived, 1) == x.parts - 1;
                if (last_one) *arrived = 0;
            }
            if (!__shfl_sync(0xffffffffu, last_one, 0)) continue;
            __threadfence();
            // of the row of this lane: maximum and sum over the pieces, four under way at a time
            auto weight = [](float2 ml, float top) {  // a NaN piece has a sum that is one, whatever its maximum
                return ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : exp2_of(ml.x - top);
            };
            float2 ml[4];
            auto four = [&](int i0) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    ml[i] = i0 + i < x.parts ? __ldcg(a.part_ml + (int64_t)x.slot(i0 + i) * TR + r0 + lane) : make_float2(-INFINITY, 0.0f);
            };
            float M = -INFINITY, L = 0.0f;
#pragma unroll 1
            for (int i0 = 0; i0 < x.parts; i0 += 4) {
                four(i0);
                const float top = fmaxf(max3(M, ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
                L *= weight(make_float2(M, 0.0f), top);
                M = top;
#pragma unroll
                for (int i = 0; i < 4; i++) L += ml[i].y * weight(ml[i], M);
            }
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            constexpr int V = D / 32, AT_ONCE = D == 256 ? 4 : 8;       // values a lane, neighbours; rows under way, of four pieces each
#pragma unroll 1
            for (int r = 0; r < rows; r += AT_ONCE) {
                float y[AT_ONCE][V] = {};
#pragma unroll 1
                for (int i0 = 0; i0 < x.parts; i0 += 4) {
                    if (x.parts > 4) four(i0);
                    float z[4][AT_ONCE][V];
#pragma unroll
                    for (int i = 0; i < 4; i++) {                       // pieces and rows past the last: the last, or what stands there, unused
                        const float* from = a.part_o + ((int64_t)x.slot(min(i0 + i, x.parts - 1)) * TR + r0 + r) * D + lane * V;
#pragma unroll
                        for (int u = 0; u < AT_ONCE; u++) {
                            if constexpr (V == 2) *(float2*)z[i][u] = __ldcg((const float2*)(from + u * D));
                            else
#pragma unroll
                                for (int e = 0; e < V; e += 4) *(float4*)(z[i][u] + e) = __ldcg((const float4*)(from + u * D + e));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float mine_w = weight(ml[i], M);
#pragma unroll
                        for (int u = 0; u < AT_ONCE; u++) {
                            const float w = __shfl_sync(0xffffffffu, mine_w, r + u);
#pragma unroll
                            for (int e = 0; e < V; e++) y[u][e] = i0 + i < x.parts ? y[u][e] + z[i][u][e] * w : y[u][e];
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++) {
                    const float f = __shfl_sync(0xffffffffu, inv, r + u);
                    const int64_t to = __shfl_sync(0xffffffffu, out_at, r + u);
                    if (r + u >= rows) continue;
#pragma unroll
                    for (int e = 0; e < V; e += 2) ((uint32_t*)(a.out + to) + lane * (V / 2))[e / 2] = pack2<T>(y[u][e] * f, y[u][e + 1] * f);
                }
            }
        }
    } else {
        at_fewer_regs();                          // (the rows' registers come from every other warp)
    }
    pf_fence_before();
    __syncthreads();
    pf_fence_after();
    if (warp == AT_MMA_WARP) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <class T> constexpr bool at_is_half = false;
template <> constexpr bool at_is_half<__half> = true;
// Pages of fewer than 16 tokens go by cp.async: a tile would be sixteen boxes and more.
constexpr int AT_LEAST_BOX = 16;
// A pool as the copy engine takes it.  False where it cannot (a stride out of its range): cp.async can.
static bool at_map(CUtensorMap* m, const Pool& p, const AttendCall& a, int dim, bool half, int rows) {
    static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess) cudaGetLastError();
        return (PFN_cuTensorMapEncodeTiled_v12000)(found == cudaDriverEntryPointSuccess ? f : nullptr);
    }();
    if (!encode || p.n_pages < 1 || p.token <= 0 || p.head <= 0 || p.page <= 0) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)dim, a.page.d, (cuuint64_t)a.heads_kv, (cuuint64_t)p.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)p.token, (cuuint64_t)p.head, (cuuint64_t)p.page};
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, step[4] = {1, 1, 1, 1};
    return encode(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, p.data, dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, class T> static cudaError_t tc(const AttendCall& a, int sm_count, cudaStream_t stream) {
    static_assert(At<D>::fixed + share_smem(kCacheSeqs, AT_THREADS) <= 227 * 1024, "the block must fit in shared memory");
    static std::atomic<uint64_t> attr_set{0};
    if (cudaError_t e = ensure_dynamic_smem(attend_tc_kernel<D, T>, (int)(At<D>::fixed + share_smem(kCacheSeqs, AT_THREADS)), attr_set)) return e;
    // setmaxnreg deals out the registers that the block was launched with: a build that launches with fewer
    // would wait for the rest for ever
    static const int regs = [] {
        cudaFuncAttributes f;
        return cudaFuncGetAttributes(&f, attend_tc_kernel<D, T>) == cudaSuccess ? f.numRegs : 0;
    }();
    if (regs * AT_THREADS < 256 * (AT_ROW_REGS + AT_OTHER_REGS)) return cudaErrorLaunchOutOfResources;
    AtMaps maps;
    maps.rows = 0;
    int rows = 128;                   // the largest power of two, up to a tile, that divides a page
    while (a.page.d % rows) rows /= 2;
    if (rows >= AT_LEAST_BOX && at_map(&maps.k, a.k, a, D, at_is_half<T>, rows) &&
        at_map(&maps.v, a.v, a, D, at_is_half<T>, rows))
        maps.rows = rows;
    count_launch();
    return launch_with(pdl_mode() == 1, stream, attend_tc_kernel<D, T>, dim3(sm_count), dim3(AT_THREADS),
                       (size_t)At<D>::fixed + share_smem(a.n_seq, AT_THREADS), a, maps);
}
cudaError_t launch_attend_tc(const AttendCall& a, int head_dim, int ggml_type, int sm_count, cudaStream_t stream) {
    const bool f16 = ggml_type == BIVMOE_F16;
    switch (head_dim) {
        case 64: return f16 ? tc<64, __half>(a, sm_count, stream) : tc<64, __nv_bfloat16>(a, sm_count, stream);
        case 128: return f16 ? tc<128, __half>(a, sm_count, stream) : tc<128, __nv_bfloat16>(a, sm_count, stream);
        default: return f16 ? tc<256, __half>(a, sm_count, stream) : tc<256, __nv_bfloat16>(a, sm_count, stream);
    }
}

}  // namespace bivmoe
