// Linear attention for prompts: 64 tokens at a time on the fifth-generation tensor cores (bf16 rows, heads of 128 x 128,
// no delta rule).
//
// With G_i the sum of a chunk's decays up to token i, S the state before the chunk, and all products turned so that a row of
// dim_v is a lane of tensor memory:
//     out_i = scale (exp(G_i) S q_i + sum_{j <= i} exp(G_i - G_j) (q_i k_j) v_j)     R = S Q^T,   N = V^T P^T
//     S    <- exp(G_63) S + sum_j exp(G_63 - G_j) v_j k_j^T                          U = W^T K,   W_j = exp(G_63 - G_j) v_j
// A thread block takes a head of a request and goes through its chunks:
//
//   warps 0-3    the state, 128 values of a row of it in a thread's registers from the first chunk to the last: exp(G) S + U
//                in f32; as bf16 into shared memory for the next chunk's R
//   warps 4-7    W^T into tensor memory, as three bf16 terms, which are W itself: the state's sums are as exact as f32
//                ones.  K is exact in bf16, so three products make U.
//   warps 8-11   out: exp(G_i) R + N
//   warps 12-13  P = Q K^T and its decays, rounded to bf16 once, into shared memory
//   warp 14      one lane issues the products
//   warp 15      brings Q, K and V by the copy engine, three chunks ahead, and works out the decays (sums in f64)
//
// V with an infinity or NaN in it would reach tokens before it (0 x infinity in N): such a place is taken out, and its row of
// out from its token on, and of the state, is NaN.
// Bytes would take 51 us for 37 requests of 2048 tokens, 4 heads (a block to an SM); it takes 80, 2.1 us a chunk: the tensor cores work a
// third of the time, issue slots half of it, and what is left is the way of a chunk from role to role.
//
// A request of many chunks may have a cluster of blocks, each with a stretch of its chunks: all but the last first find what
// their stretch adds to the state (U alone: K and V are read twice), then hand the state on through distributed shared memory,
// a multiplication and an addition each, and then every block does its stretch's outputs from the state it was given.
#include <stddef.h>

#include "common.cuh"
#include "launch.cuh"
#include "linear_tc.cuh"

namespace bivmoe {

namespace {

constexpr int kThreads = 512, kStages = 3, kRing = 8;
constexpr int kStateRegs = 208, kOtherRegs = 96;
static_assert((kStateRegs + 3 * kOtherRegs) * 128 <= 65536, "setmaxnreg would wait for registers that nobody gives");
constexpr int kStage = kQK + kV, kState = 2 * kHalf, kP = C * 128;
// tensor memory: U, R, N, Q K^T, and W twice
constexpr uint32_t kAtU = 0, kAtR = 128, kAtN = 192, kAtQK = 256, kAtW = 320;
enum { SITE_STATE = 41, SITE_W, SITE_OUT, SITE_P, SITE_MMA, SITE_COPY };

struct alignas(16) Decays {                          // of a chunk
    float log2[C], left[C], upto[C];                 // G_j log2(e), exp(G_63 - G_j), exp(G_j)
    float whole;                                     // exp(G_63)
    double sum;                                      // of all the decays of the stretch so far
    uint8_t bad[D];                                  // the first token whose value of v is not finite, or 255
};
struct Head {
    uint64_t full[kStages], empty[kStages], known[kRing], qk_full, qk_free, p_full[2], w_full[kRing], w_free[2], u_full, u_free, s_full, r_done,
        n_full, o_free, out_done, given, read, drained;
    uint32_t tmem;
    int abort;
    Decays ring[kRing];
};
static_assert(offsetof(Head, ring) % 16 == 0 && sizeof(Decays) % 16 == 0 && offsetof(Decays, left) % 16 == 0, "read by 8 and 16 bytes");
constexpr int kHeadBytes = (sizeof(Head) + 1023) / 1024 * 1024;
constexpr int kSmem = kHeadBytes + kStages * kStage + 2 * kState + kP;   // (the state handed on between blocks is f32)
static_assert(kSmem <= 227 * 1024 && kP + 4 * 4096 <= kState, "the block must fit in shared memory");

struct Maps { CUtensorMap q, k, v; };

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {     // the same place of another block of the cluster
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__global__ void __launch_bounds__(kThreads, 1) linear_chunks_kernel(const __grid_constant__ LinearCall c, const __grid_constant__ Maps maps) {
    extern __shared__ __align__(1024) uint8_t sm[];
    Head& H = *(Head*)sm;
    const uint32_t stages = pf_smem(sm) + kHeadBytes, state = stages + kStages * kStage, weights = state + 2 * kState;
    // P of odd chunks, and the outputs on their way out, lie in the second half of what a state in f32 is handed over in: there are
    // none before the first R
    auto weights_of = [&](int j) { return j & 1 ? state + kState : weights; };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 416) {
        for (int i = 0; i < kStages; i++) { pf_bar_init(&H.full[i], 1); pf_bar_init(&H.empty[i], 1); }
        for (int i = 0; i < kRing; i++) { pf_bar_init(&H.known[i], 1); pf_bar_init(&H.w_full[i], 4); }
        for (int i = 0; i < 2; i++) pf_bar_init(&H.w_free[i], 1);
        for (uint64_t* one : {&H.qk_full, &H.u_full, &H.r_done, &H.n_full, &H.drained}) pf_bar_init(one, 1);
        for (uint64_t* four : {&H.u_free, &H.s_full, &H.o_free, &H.out_done, &H.read}) pf_bar_init(four, 4);
        for (uint64_t* two : {&H.qk_free, &H.p_full[0], &H.p_full[1]}) pf_bar_init(two, 2);
        pf_bar_init(&H.given, 128);
        H.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 480) prefetch_maps(maps.q, maps.k, maps.v);
    pdl_enter();
    const int blocks = (int)cluster_size(), rank = (int)cluster_rank();
    const int work = blockIdx.x / blocks, h = work % c.n_head, b = request_at(c, work / c.n_head);
    const LinearSeq seq = linear_seq(c, b);
    const bool mine = slot_taken(c, b, tid, kThreads);
    if (!seq.n) return;                              // the whole cluster
    // the state is asked for before anything else
    const int64_t at = (int64_t)h * c.head + (int64_t)(warp * 32) * D;           // a state warp's rows
    const uint32_t room = state + (warp & 3) * (32 * D * 4);                     // and where they stand while they are handed over
    if (warp < 4 && !rank && seq.from) ask_for_state<32>(seq.from + at, room, 0);
    if (warp == 14) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pf_smem(&H.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pf_fence_before();
    const bool taken = __syncthreads_or(mine);
    if (blocks > 1) cluster_meet();
    pf_fence_after();
    const uint32_t tmem = H.tmem;
    auto give_up = [&](int site) {
        if (lane == 0) {
            atomicExch(c.status, site);
            *(volatile int*)&H.abort = 1;
        }
    };
    // Where a chunk's values are not finite comes from the weights' warps, its decays from the copying one, which those have waited for: their
    // word, `w_full`, is asked for together with the end of the product that a role waits for.  (A place of the ring is told again eight
    // chunks on, and no role's own chunk is left behind by as many: behind its product the phase that ended last is the chunk's.  That is
    // so for roles, too, that sit the first pass out and have not followed the ring, of which the parity alone would say nothing.  As a wait of its
    // own, and one for `known`, a prompt of 8192 tokens and 32 heads took 140 us and not 132.)
    // this block's chunks; those that it goes through twice
    const int chunks = (seq.n + C - 1) / C, c0 = (int)((int64_t)chunks * rank / blocks), own = (int)((int64_t)chunks * (rank + 1) / blocks) - c0;
    const int twice = rank + 1 < blocks ? own : 0;

    if (warp < 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kStateRegs));
        // ---- the state
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        float s[D];
#pragma unroll
        for (int i = 0; i < D; i++) s[i] = 0.0f;
        bool ok = true;
        for (int k = 0;; k++) {
            if (k == twice) {
                // the state that the stretch starts from: its own place if the block is the first, else as the one before
                // hands it on; and handed on to the one behind
                if (rank && !wait_here<true>(&H.given, 0, &H)) { ok = false; break; }
                const float whole = twice ? expf((float)H.ring[(twice - 1) % kRing].sum) : 1.0f;
                const bool more = rank + 1 < blocks, has = rank || (seq.from && !taken);
                wait_for_state();
                auto piece = [&](int p) { return has ? lds128(state_piece(room, lane, p)) : make_uint4(0, 0, 0, 0); };
                if (more) {
                    const uint32_t to = in_block(room, rank + 1);
#pragma unroll
                    for (int p = 0; p < D / 4; p++) {
                        const uint4 x = piece(p);
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(state_piece(to, lane, p)),
                                     "f"(fmaf(whole, __uint_as_float(x.x), s[4 * p])), "f"(fmaf(whole, __uint_as_float(x.y), s[4 * p + 1])),
                                     "f"(fmaf(whole, __uint_as_float(x.z), s[4 * p + 2])), "f"(fmaf(whole, __uint_as_float(x.w), s[4 * p + 3])) : "memory");
                    }
                }
#pragma unroll
                for (int p = 0; p < D / 4; p++) {
                    const uint4 x = piece(p);
                    s[4 * p] = __uint_as_float(x.x); s[4 * p + 1] = __uint_as_float(x.y); s[4 * p + 2] = __uint_as_float(x.z); s[4 * p + 3] = __uint_as_float(x.w);
                }
                if (more)
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_block(pf_smem(&H.given), rank + 1)) : "memory");
                // all warps have read theirs before its place takes the state for the first R
                __syncwarp();
                arrive_warp(&H.read);
                if (!wait_here(&H.read, 0, &H)) { ok = false; break; }
            }
            if (k == twice + own) break;
            if (k >= twice) {
                // the state before the chunk for its R, rounded to bf16 as the chunk's P is: each is off by half a step of
                // the outputs' own type, in values that differ from one another
                if (k > twice && !wait_here(&H.r_done, (k - twice - 1) & 1, &H)) { ok = false; break; }
#pragma unroll
                for (int p = 0; p < 16; p++) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = narrow2(s[8 * p + 2 * i], s[8 * p + 2 * i + 1], BIVMOE_BF16);
                    sts128(state + (p >> 3) * kHalf + tid * 128 + (((p ^ tid) & 7) << 4), w[0], w[1], w[2], w[3]);
                }
                fence_async();
                __syncwarp();
                arrive_warp(&H.s_full);
            }
            // the chunk's sum joins it
            if (!wait_told_here(&H.u_full, k & 1, &H.w_full[k % kRing], (k / kRing) & 1, &H)) { ok = false; break; }
            pf_fence_after();
            const Decays& dec = H.ring[k % kRing];
            const float by = dec.bad[tid] == 255 ? dec.whole : __int_as_float(0x7fffffff);   // (NaN: so becomes the row)
            const f32x2 by2 = pk(by, by);
#pragma unroll
            for (int e = 0; e < D; e += 32) {
                int u[32];
                pf_tmem_ld32(tmem + kAtU + e + lanes, u);
                pf_tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const f32x2 x = fma2(by2, pk(s[e + i], s[e + i + 1]), pk(__int_as_float(u[i]), __int_as_float(u[i + 1])));
                    s[e + i] = lo_of(x);
                    s[e + i + 1] = hi_of(x);
                }
            }
            pf_fence_before();
            __syncwarp();
            arrive_warp(&H.u_free);
        }
        // (the last products have read the state and P, and the last outputs have left, when the state's place is taken for its way out; the
        // outputs' word first, since these warps have not followed n_full and its parity alone says nothing)
        if (ok && rank + 1 == blocks && seq.to && !taken) {
            if (wait_here(&H.out_done, 0, &H) && wait_here(&H.n_full, (own - 1) & 1, &H)) store_state(s, seq.to + at, room, 0);
            else ok = false;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");      // (where a wait gave up before it was looked at)
        if (!ok) give_up(SITE_STATE);
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        // ---- W: turned by ldmatrix, so that a register holds two tokens' values of a row of dim_v, as tensor memory wants them
        const int quarter = warp & 3;                // 32 rows of dim_v
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        for (int k = 0; k < twice + own; k++) {
            if (!wait_warp(&H.known[k % kRing], (k / kRing) & 1, &H) || !wait_warp(&H.full[k % kStages], (k / kStages) & 1, &H) ||
                !wait_warp(&H.w_free[k & 1], ((k >> 1) & 1) ^ 1, &H)) {
                give_up(SITE_W);
                break;
            }
            pf_fence_after();
            Decays& dec = H.ring[k % kRing];
            const uint32_t v = stages + (k % kStages) * kStage + kQK + (quarter >> 1) * (C * 128), to = tmem + kAtW + (k & 1) * 96 + lanes;
            dec.bad[quarter * 32 + lane] = 255;
#pragma unroll 1
            for (int again = 0; again < 2; again++) {
                uint32_t odd = 0;
#pragma unroll 1
                for (int part = 0; part < 4; part++) {        // 16 rows, 32 tokens
                    const int r16 = part >> 1, j0 = (part & 1) * 32;
                    uint32_t w[3][8];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        // matrices of 8 tokens x 8 rows: tokens j0 + 16 e + 0..7 and 8..15, of each the two groups of eight rows
                        const int row = j0 + 16 * e + 8 * (lane >> 4) + (lane & 7), piece = (quarter & 1) * 4 + r16 * 2 + (lane >> 3 & 1);
                        uint32_t x[4];
                        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(v + row * 128 + (((piece ^ row) & 7) << 4)) : "memory");
#pragma unroll
                        for (int i = 0; i < 4; i++) {         // i >> 1: the tokens' eight, i & 1: the rows'
                            asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(odd) : "r"(x[i]), "r"(0u));
                            const float2 left = *(const float2*)&dec.left[j0 + 16 * e + 8 * (i >> 1) + 2 * (lane & 3)];
                            f32x2 z = mul2(pk(__uint_as_float(x[i] << 16), __uint_as_float(x[i] & 0xffff0000u)), pk(left.x, left.y));
                            w[0][4 * e + i] = bf16_term(z);
                            w[1][4 * e + i] = bf16_term(z);
                            w[2][4 * e + i] = last_term(z);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 3; i++) tmem_st_16x4(to + ((uint32_t)(r16 * 16) << 16) + 32 * i + j0 / 2, w[i]);
                }
                if (again || !__any_sync(0xffffffffu, odd != 0)) break;
                // Something is not finite: taken out, its row's first token noted.
                uint32_t bad = 255;
#pragma unroll 1
                for (int j = C - 1; j >= 0; j--) {
                    const uint32_t a = v + j * 128 + (((((quarter & 1) * 4 + (lane >> 3)) ^ j) & 7) << 4) + (lane & 7) * 2;
                    if ((lds16(a) & 0x7f80u) == 0x7f80u) {
                        bad = j;
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"((uint16_t)0) : "memory");
                    }
                }
                dec.bad[quarter * 32 + lane] = (uint8_t)bad;
                fence_async();
                __syncwarp();                                 // what a lane has taken out, before another loads it
                if (!__any_sync(0xffffffffu, bad != 255)) break;
            }
            wait_st();
            pf_fence_before();
            __syncwarp();
            arrive_warp(&H.w_full[k % kRing]);
        }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        // ---- out
        const uint32_t tile = state + kState + kP + (warp & 3) * 4096;           // (there is no handed over state any more)
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        uint8_t* out = c.out.data + (int64_t)(seq.first + c0 * C) * c.out.token + h * c.out.head + (warp & 3) * 64;
        for (int j = 0; j < own; j++, out += C * c.out.token) {
            const int k = twice + j, n = min(C, seq.n - (c0 + j) * C);
            if (!wait_told(&H.n_full, j & 1, &H.w_full[k % kRing], (k / kRing) & 1, &H)) { give_up(SITE_OUT); break; }
            pf_fence_after();
            const Decays& dec = H.ring[k % kRing];
            write_out(tmem + kAtR + lanes, tmem + kAtN + lanes, dec.upto, c.scale, [&](int r) { return (int)dec.bad[(warp & 3) * 32 + r]; },
                      tile, out, c.out.token, n, &H.o_free);
        }
        arrive_warp(&H.out_done);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp < 14) {
            // ---- P: a token's row to a thread
            const int r = tid - 384;
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            for (int j = 0; j < own; j++) {
                const int k = twice + j;
                if (!wait_told(&H.qk_full, j & 1, &H.known[k % kRing], (k / kRing) & 1, &H)) { give_up(SITE_P); break; }
                pf_fence_after();
                // (two P: this one's place was read by the product two chunks ago, which ended before this Q K^T did)
                weights_row(tmem + kAtQK + lanes, H.ring[k % kRing].log2, r, weights_of(j) + r * 128, &H.qk_free);
                fence_async();
                __syncwarp();
                arrive_warp(&H.p_full[j & 1]);
            }
        } else if (warp == 14) {
            // ---- products
            if (pf_elect()) {
                bool ok = true;
                auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = ok && wait_one(bar, parity, &H); };
                auto stage = [&](int k) { return stages + (k % kStages) * kStage; };
                auto u_of = [&](int k) {
                    wait(&H.full[k % kStages], (k / kStages) & 1);
                    wait(&H.w_full[k % kRing], (k / kRing) & 1);
                    if (k) wait(&H.u_free, (k - 1) & 1);
                    if (!ok) return;
                    pf_fence_after();
                    fence_async();
                    const uint32_t w = tmem + kAtW + (k & 1) * 96, at = stage(k) + C * 128;
                    const uint64_t key = desc_mn(at, kHalf);
#pragma unroll 1
                    for (int i = 0; i < 3; i++)          // the smallest terms first
#pragma unroll
                        for (int e = 0; e < C / 16; e++)
                            mma_ts(tmem + kAtU, w + 32 * (2 - i) + 8 * e, key + (2048 >> 4) * e, idesc(D, false, true), i || e);
                    pf_commit(&H.u_full);
                    pf_commit(&H.w_free[k & 1]);
                };
                auto qk_of = [&](int k, int j) {
                    wait(&H.full[k % kStages], (k / kStages) & 1);
                    wait(&H.known[k % kRing], (k / kRing) & 1);      // (a chunk that is not full has been cleared)
                    if (j) wait(&H.qk_free, (j - 1) & 1);
                    if (!ok) return;
                    pf_fence_after();
                    fence_async();
                    const uint64_t both = pf_desc_sw128(stage(k)), key = pf_desc_sw128(stage(k) + C * 128);
#pragma unroll 1
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            pf_mma_bf16(tmem + kAtQK, both + half * (kHalf >> 4) + 2 * e, key + half * (kHalf >> 4) + 2 * e, idesc(C, false, false), half || e);
                    pf_commit(&H.qk_full);
                };
                for (int k = 0; k < twice && ok; k++) {
                    u_of(k);
                    if (ok) pf_commit(&H.empty[k % kStages]);
                }
                if (own && ok) qk_of(twice, 0);
                for (int j = 0; j < own && ok; j++) {
                    const int k = twice + j;
                    u_of(k);
                    wait(&H.s_full, j & 1);
                    if (j) wait(&H.o_free, (j - 1) & 1);
                    if (!ok) break;
                    pf_fence_after();
                    fence_async();
                    const uint64_t before = pf_desc_sw128(state), query = pf_desc_sw128(stage(k));
#pragma unroll 1
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            pf_mma_bf16(tmem + kAtR, before + half * (kHalf >> 4) + 2 * e, query + half * (kHalf >> 4) + 2 * e, idesc(C, false, false), half || e);
                    pf_commit(&H.r_done);
                    // the next chunk's Q K^T, if it is here; else after this one's last product, with whose end a place for copies
                    // becomes free
                    bool asked = j + 1 == own;
                    if (!asked && pf_bar_try(&H.full[(k + 1) % kStages], ((k + 1) / kStages) & 1)) {
                        qk_of(k + 1, j + 1);
                        asked = true;
                    }
                    wait(&H.p_full[j & 1], (j >> 1) & 1);
                    if (!ok) break;
                    pf_fence_after();
                    fence_async();
                    const uint64_t value = desc_mn(stage(k) + kQK, C * 128), weight = pf_desc_sw128(weights_of(j));
#pragma unroll
                    for (int e = 0; e < C / 16; e++)
                        pf_mma_bf16(tmem + kAtN, value + (2048 >> 4) * e, weight + 2 * e, idesc(C, true, false), e != 0);
                    pf_commit(&H.n_full);
                    pf_commit(&H.empty[k % kStages]);
                    if (!asked) qk_of(k + 1, j + 1);
                }
                if (!ok) {
                    atomicExch(c.status, SITE_MMA);
                    *(volatile int*)&H.abort = 1;
                }
            }
            __syncwarp();
            // nothing is in flight when the block ends, whatever ended the loops
            if (pf_elect()) pf_commit(&H.drained);
            __syncwarp();
            pf_bar_wait(&H.drained, 0);
            __syncwarp();
        } else {
            // ---- copies and decays: two tokens to a lane
            const int hq = h / c.group;
            double all = 0.0;
            int copies = 0;
            auto chunk_of = [&](int k) { return c0 + (k < twice ? k : k - twice); };
            auto decays_of = [&](int k, float (&g)[2]) {
                const int n = k < twice + own ? seq.n - chunk_of(k) * C : 0, token = seq.first + chunk_of(k) * C;
#pragma unroll
                for (int i = 0; i < 2; i++) g[i] = lane + 32 * i < n ? c.decay[(int64_t)(token + lane + 32 * i) * c.decay_stride + h] : 0.0f;
            };
            float next[2];
            decays_of(0, next);
            auto copy = [&](int k) {
                const bool alone = k < twice;        // K and V alone
                uint64_t* full = &H.full[k % kStages];
                const uint32_t at = stages + (k % kStages) * kStage;
                const int token = seq.first + chunk_of(k) * C;
                copies++;
                if (lane == 0) {
                    pf_bar_expect_tx(full, alone ? 4 * C * 128 : 6 * C * 128);
                    for (int half = 0; half < 2; half++) {
                        box(at + half * kHalf + C * 128, &maps.k, half * 64, hq, token, full);
                        box(at + kQK + half * (C * 128), &maps.v, half * 64, h, token, full);
                        if (!alone) box(at + half * kHalf, &maps.q, half * 64, hq, token, full);
                    }
                }
                __syncwarp();
            };
            for (int k = 0; k < kStages && k < twice + own; k++) copy(k);
            for (int k = 0; k < twice + own; k++) {
                const int n = min(C, seq.n - chunk_of(k) * C);
                if (k == twice) all = 0.0;
                // the copies before the decays, whose next ones are on their way meanwhile
                if (k >= kStages) {
                    if (!wait_warp(&H.empty[k % kStages], ((k / kStages) & 1) ^ 1, &H)) { give_up(SITE_COPY); break; }
                    copy(k);
                }
                const float g[2] = {clamp_decay(next[0]), clamp_decay(next[1])};
                decays_of(k + 1, next);
                double x[2];
                const double whole = sums_of_decays(g, x);
                all += whole;
                Decays& dec = H.ring[k % kRing];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int j = lane + 32 * i;
                    dec.log2[j] = (float)(x[i] * 1.4426950408889634);
                    dec.left[j] = j < n ? expf((float)(whole - x[i])) : 0.0f;
                    dec.upto[j] = expf((float)x[i]);
                }
                if (lane == 0) {
                    dec.whole = expf((float)whole);
                    dec.sum = all;
                }
                if (n < C) {
                    if (!wait_warp(&H.full[k % kStages], (k / kStages) & 1, &H)) { give_up(SITE_COPY); break; }
                    clear_rows(stages + (k % kStages) * kStage, n);
                }
                __syncwarp();
                arrive_warp(&H.known[k % kRing]);
            }
            // no copy is under way when the block ends, whatever ended the loop
            if (copies) wait_for_last_fills<kStages, 1>((uint32_t)(copies - 1), (uint32_t)copies, [&](uint32_t slot, uint32_t parity) { pf_bar_wait(&H.full[slot], parity); });
            __syncwarp();
        }
    }
    pf_fence_before();
    __syncthreads();
    pf_fence_after();
    if (warp == 14) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (blocks > 1) cluster_meet();                  // nobody is written to, or waited for, that has left
}

int g_regs = 0;                                      // a thread's, as built

constexpr int kClusters = 3;                         // clusters of two, four and eight blocks
int g_clusters[kClusters + 1];                       // that run at once
void set_launch(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, unsigned blocks, unsigned cluster) {
    cfg->gridDim = dim3(blocks);
    cfg->blockDim = dim3(kThreads);
    cfg->dynamicSmemBytes = kSmem;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg->attrs = attr;
    cfg->numAttrs = cluster > 1 ? 1 : 0;
}

}  // namespace

cudaError_t linear_chunks_attributes() {
    cudaFuncAttributes f;
    cudaError_t e = cudaFuncGetAttributes(&f, linear_chunks_kernel);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(linear_chunks_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess) g_regs = f.numRegs;
    for (int i = 1; i <= kClusters && e == cudaSuccess; i++) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[1];
        set_launch(&cfg, attr, 1 << i, 1 << i);
        e = cudaOccupancyMaxActiveClusters(&g_clusters[i], linear_chunks_kernel, &cfg);
    }
    return e;
}

// Blocks to a request and head: as many as run at once, if each has some chunks.  us with one, two, four and eight blocks: 32 heads of
// 512 tokens 25, 27, 30; of 1024 41, 40, 37; of 8192 257, 223, 132; 8 heads of 2048 71, 66, 48, 52; of 8192 253, 217, 126, 92.  Where
// they do not fit they take turns: 16 heads of 8192 tokens by eight blocks each 183 us, 64 of 1024 by four 70 and not 41.
static int cluster_of(const LinearCall& c, int max_new) {
    const int64_t work = (int64_t)c.n_seq * c.n_head;
    const int chunks = (max_new + C - 1) / C;
    int i = 0;
    while (i < kClusters && work <= g_clusters[i + 1] && chunks >= (i == 2 ? 64 : 16)) i++;
    return 1 << i;
}

bool launch_linear_chunks(const LinearCall& c, int max_new, cudaStream_t stream, cudaError_t* e) {
    // setmaxnreg deals out the registers that the block was launched with: a build that launches with fewer would wait for ever
    if (g_regs * 4 < kStateRegs + 3 * kOtherRegs) return false;
    Maps maps;
    if (!map_rows(&maps.q, c.q, c.n_head / c.group, c.n_tokens) || !map_rows(&maps.k, c.k, c.n_head / c.group, c.n_tokens) ||
        !map_rows(&maps.v, c.v, c.n_head, c.n_tokens))
        return false;
    const int blocks = cluster_of(c, max_new);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    set_launch(&cfg, attr, (unsigned)(c.n_seq * c.n_head * blocks), (unsigned)blocks);
    cfg.stream = stream;
    count_launch();
    *e = cudaLaunchKernelEx(&cfg, linear_chunks_kernel, c, maps);
    return true;
}

}  // namespace bivmoe
