// Linear attention with the delta rule for prompts: 64 tokens at a time on the fifth-generation tensor cores (bf16 rows, heads of
// 128 x 128).
//
// Within a chunk, with G_i the sum of the decays up to token i and S the state before it, a token's own addition is u_i k_i^T with
//     u_i = beta_i (v_i - exp(G_i) S k_i - sum_{j < i} exp(G_i - G_j) (k_i k_j) u_j)
// that is, (I + L) u = rhs with L_ij = beta_i exp(G_i - G_j) (k_i k_j) below the diagonal and rhs_i = beta_i (v_i - exp(G_i) S k_i).
// T = (I + L)^-1 needs K and the decays alone, so that it is made while the chunk before is still at work, and then
//     u = T rhs,    out_i = scale (exp(G_i) S q_i + sum_{j <= i} exp(G_i - G_j) (q_i k_j) u_j),    S <- exp(G_63) S + sum_j exp(G_63 - G_j) u_j k_j^T
// All products are turned so that a row of dim_v is a lane of tensor memory.  A thread block takes a head of a request and goes through
// its chunks, each of them a chain of products and of what stands between them:
//
//   warps 0-7    the chain: the state, 64 values of a row of it in a thread's registers, as three bf16 terms, which are the state itself, for
//                S [Q; K]; rhs from S k and V, in three terms; u from the product with T, in two for the outputs, and as W, times
//                its decay to the chunk's end, in three for the state; exp(G) S + U in f32
//   warps 8-11   the outputs
//   warps 12-13  P = Q K^T and its decays, rounded to bf16 once
//   warps 14, 15, 18, 19  L from K K^T, T in f32; in three terms
//   warp 16      one lane issues the products;  warp 17: copies and decays
//
// Not bytes bound it but these steps.  A chunk takes 13400 clocks (37 requests of 2048 tokens, 4 heads, a block to an SM: 224 us, bytes alone
// 51), of which the tensor cores work a quarter: T's own steps take some 11000, the chain's, which T(k + 1) runs beside, 9000.
// (With the chain in four warps and the outputs in it 242 us; with eight warps for T 230.)
//
// Places that are not finite would reach tokens before their own through a product with zeros: they are taken out of rhs and u, and their
// row of out from their token on, and of the state, is NaN.
#include <stddef.h>

#include "common.cuh"
#include "launch.cuh"
#include "linear_tc.cuh"

namespace bivmoe {

namespace {

constexpr int kChain = 256, kThreads = kChain + 384, kStages = 2, kRing = 4;
constexpr int kChainRegs = 144, kOtherRegs = 64;
static_assert(kChain * kChainRegs + (kThreads - kChain) * kOtherRegs <= 65536, "setmaxnreg would wait for registers that nobody gives");
constexpr int kStage = kQK + kV, kTerm = 2 * kHalf, kP = C * 128;
// L turned, T, T turned within its blocks of 32, a product: rows of these many floats, so that lanes apart by rows meet banks apart
constexpr int kL = 68, kT = 68, kTurned = 36, kBetween = 36;
constexpr int kWork = (C * kL + 32 * kBetween) * 4;
// tensor memory: the state's first two terms, for each half of dim_k, later U; S Q^T and S K^T, and where the latter stood u in two terms; T rhs, later N;
// Q K^T and K K^T; rhs, later W
constexpr uint32_t kAtU = 0, kAtR = 128, kAtSK = 192, kAtX = 256, kAtQK = 320, kAtW = 384;
enum { SITE_CHAIN = 51, SITE_OUT, SITE_P, SITE_T, SITE_MMA, SITE_COPY };

struct alignas(16) Decays {                          // of a chunk
    float log2[C], left[C], upto[C], beta[C];        // G_j log2(e), exp(G_63 - G_j), exp(G_j)
    float minus[2][C];                               // -G_j log2(e) as an f32 number and what that leaves of it
    float whole;                                     // exp(G_63)
    int odd_row;                                     // the first row of L that is not finite, or C
    int bad[D];                                      // the first token whose u is not finite, or C
};
struct Head {
    uint64_t full[kStages], full_v[kStages], spent[kStages], empty[kStages], known[kRing], qk_full[2], qk_free, p_full, t_full, s_full, rk_full, rhs_full, x_full[2], w_full,
        u_full, n_full, o_free, read, drained;
    uint32_t tmem;
    int abort;
    alignas(16) Decays ring[kRing];
};
constexpr int kHeadBytes = (sizeof(Head) + 1023) / 1024 * 1024;
constexpr int kSmem = kHeadBytes + kStages * kStage + 2 * kTerm + 4 * kP + kWork;       // (a state on its way in or out takes two terms' room)
static_assert(kSmem <= 227 * 1024 && (C * kT + C * kTurned) * 4 <= kTerm, "the block must fit in shared memory");
static_assert(offsetof(Head, ring) % 16 == 0 && sizeof(Decays) % 16 == 0 && offsetof(Decays, upto) % 16 == 0 && offsetof(Decays, minus) % 16 == 0, "read by 16 bytes");

struct Maps { CUtensorMap q, k, v; };

// Four warps meet, at a barrier that knows no end of waiting: none of them waits for anything else in such a way, or leaves alone.
__device__ __forceinline__ void meet_four() { asm volatile("barrier.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool all_of_four(bool mine) {
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(all) : "r"((uint32_t)mine) : "memory");
    return all != 0;
}
// Four rows of a column of a product of n inner values: `left` turned (a row's four neighbours), `right` from the column on.
__device__ __forceinline__ float4 product4(const float* left, int left_row, const float* right, int right_row, int n) {
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int j = 0; j < n; j++) {
        const float4 l = *(const float4*)(left + j * left_row);
        const float x = right[j * right_row];
        y.x = fmaf(l.x, x, y.x);
        y.y = fmaf(l.y, x, y.y);
        y.z = fmaf(l.z, x, y.z);
        y.w = fmaf(l.w, x, y.w);
    }
    return y;
}

// A tile of 16 x 16, to a warp, of a product of 32 inner values, in f32 by bf16 terms, the smallest products of them first: `left` turned.
__device__ __forceinline__ void tile_product(const float* left, int left_row, const float* right, int right_row, float* into, int into_row, float sign) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c2 = 2 * (lane & 3);
    float y[2][4] = {};
#pragma unroll 1
    for (int k0 = 0; k0 < 32; k0 += 16) {
        uint32_t a[3][4], b[3][2][2];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float* at = left + (k0 + c2 + 8 * (q >> 1)) * left_row + g + 8 * (q & 1);
            f32x2 x = pk(at[0], at[left_row]);
            a[0][q] = bf16_term(x);
            a[1][q] = bf16_term(x);
            a[2][q] = last_term(x);
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float* at = right + (k0 + c2 + 8 * (q & 1)) * right_row + g + 8 * (q >> 1);
            f32x2 x = pk(at[0], at[right_row]);
            b[0][q >> 1][q & 1] = bf16_term(x);
            b[1][q >> 1][q & 1] = bf16_term(x);
            b[2][q >> 1][q & 1] = last_term(x);
        }
#pragma unroll
        for (int i = 0; i < 6; i++) {
            const int s = i == 0 ? 0 : i == 1 ? 1 : i == 2 ? 2 : i == 3 ? 1 : 0, t = i == 0 ? 2 : i == 1 || i == 4 ? 1 : 0;
#pragma unroll
            for (int n = 0; n < 2; n++)
                asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                             : "+f"(y[n][0]), "+f"(y[n][1]), "+f"(y[n][2]), "+f"(y[n][3])
                             : "r"(a[s][0]), "r"(a[s][1]), "r"(a[s][2]), "r"(a[s][3]), "r"(b[t][n][0]), "r"(b[t][n][1]));
        }
    }
#pragma unroll
    for (int n = 0; n < 2; n++) {
        *(float2*)&into[g * into_row + 8 * n + c2] = make_float2(sign * y[n][0], sign * y[n][1]);
        *(float2*)&into[(g + 8) * into_row + 8 * n + c2] = make_float2(sign * y[n][2], sign * y[n][3]);
    }
}

__global__ void __launch_bounds__(kThreads, 1) linear_delta_kernel(const __grid_constant__ LinearCall c, const __grid_constant__ Maps maps) {
    extern __shared__ __align__(1024) uint8_t sm[];
    Head& H = *(Head*)sm;
    const uint32_t stages = pf_smem(sm) + kHeadBytes, state = stages + kStages * kStage, weights = state + 2 * kTerm, inverse = weights + kP;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == kThreads - 32) {
        for (int i = 0; i < kStages; i++) {
            for (uint64_t* one : {&H.full[i], &H.full_v[i], &H.spent[i]}) pf_bar_init(one, 1);
            pf_bar_init(&H.empty[i], 4);
        }
        for (int i = 0; i < kRing; i++) pf_bar_init(&H.known[i], 1);
        for (uint64_t* one : {&H.qk_full[0], &H.qk_full[1], &H.rk_full, &H.x_full[0], &H.x_full[1], &H.u_full, &H.n_full, &H.drained}) pf_bar_init(one, 1);
        for (uint64_t* four : {&H.t_full, &H.o_free}) pf_bar_init(four, 4);
        for (uint64_t* eight : {&H.s_full, &H.rhs_full, &H.w_full, &H.read}) pf_bar_init(eight, 8);
        pf_bar_init(&H.p_full, 2);
        pf_bar_init(&H.qk_free, 6);
        H.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 17 * 32) prefetch_maps(maps.q, maps.k, maps.v);
    pdl_enter();
    const int h = blockIdx.x % c.n_head, b = request_at(c, blockIdx.x / c.n_head);
    const LinearSeq seq = linear_seq(c, b);
    const bool mine = slot_taken(c, b, tid, kThreads);
    if (!seq.n) return;                              // the whole block
    // the state is asked for before anything else
    const int quarter = warp & 3, side = warp >> 2;                              // 32 rows of dim_v; of the chain, half of dim_k, and of the tokens
    const int64_t at = (int64_t)h * c.head + (int64_t)(quarter * 32) * D;
    const uint32_t room = state + quarter * (32 * D * 4);                        // where the rows stand on their way in and out
    if (warp < 8 && seq.from) ask_for_state<16>(seq.from + at, room, side * 16);
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pf_smem(&H.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pf_fence_before();
    const bool taken = __syncthreads_or(mine);
    pf_fence_after();
    const uint32_t tmem = H.tmem, lanes = (uint32_t)((warp & 3) * 32) << 16;
    auto give_up = [&](int site) {
        if (lane == 0) {
            atomicExch(c.status, site);
            *(volatile int*)&H.abort = 1;
        }
    };
    const int chunks = (seq.n + C - 1) / C;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kChainRegs));
        // ---- the chain.  In rhs and u, a register of two tokens' values of a row: as ldmatrix turns V, as tensor memory's 16-lane loads
        // leave them, and as its stores want them.
        const bool has = seq.from && !taken;
        float s[D / 2];
        wait_for_state();
#pragma unroll
        for (int p = 0; p < D / 8; p++) {
            const uint4 x = has ? lds128(state_piece(room, lane, side * 16 + p)) : make_uint4(0, 0, 0, 0);
            s[4 * p] = __uint_as_float(x.x); s[4 * p + 1] = __uint_as_float(x.y); s[4 * p + 2] = __uint_as_float(x.z); s[4 * p + 3] = __uint_as_float(x.w);
        }
        // all warps have read theirs before the places take the state's terms
        __syncwarp();
        arrive_warp(&H.read);
        bool ok = wait_here(&H.read, 0, &H);
        const int row = quarter * 32 + lane, j0 = side * 32;
        for (int k = 0; k < chunks && ok; k++) {
            // Three terms, which are the state itself: two into the columns that this half's U will take, which have been read, the third
            // into shared memory (whose readers ended before the last U).
#pragma unroll
            for (int e = 0; e < D / 2; e += 32) {
                uint32_t hi[16], mid[16];
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    uint32_t lo[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        f32x2 x = pk(s[e + 8 * p + 2 * i], s[e + 8 * p + 2 * i + 1]);
                        hi[4 * p + i] = bf16_term(x);
                        mid[4 * p + i] = bf16_term(x);
                        lo[i] = last_term(x);
                    }
                    sts128(state + side * kHalf + row * 128 + (((e / 8 + p ^ row) & 7) << 4), lo[0], lo[1], lo[2], lo[3]);
                }
                tmem_st16(tmem + kAtU + 64 * side + e / 2 + lanes, hi);
                tmem_st16(tmem + kAtU + 64 * side + 32 + e / 2 + lanes, mid);
            }
            wait_st();
            pf_fence_before();
            fence_async();
            __syncwarp();
            arrive_warp(&H.s_full);
            if (!wait_here(&H.known[k % kRing], (k / kRing) & 1, &H) || !wait_here(&H.full_v[k % kStages], (k / kStages) & 1, &H) ||
                !wait_here(&H.rk_full, k & 1, &H)) {
                ok = false;
                break;
            }
            pf_fence_after();
            Decays& dec = H.ring[k % kRing];
            int* bad = dec.bad + quarter * 32;
            const uint32_t v = stages + (k % kStages) * kStage + kQK + (quarter >> 1) * (C * 128);
            // takes a value out that is not finite: token j of row r
            auto clean = [&](float& x, int r, int j) {
                if (!(fabsf(x) <= 3.402823466e38f)) {
                    atomicMin(&bad[r], j);
                    x = 0.0f;
                }
            };
#pragma unroll 1
            for (int r16 = 0; r16 < 2; r16++) {               // 16 rows, 32 tokens
                const uint32_t half = (uint32_t)(r16 * 16) << 16;
                int x[16];
                pf_tmem_ld_16x8<4>(tmem + kAtSK + j0 + lanes + half, x);
                uint32_t y[8], w[3][8];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int row = j0 + 16 * e + 8 * (lane >> 4) + (lane & 7), piece = (quarter & 1) * 4 + r16 * 2 + (lane >> 3 & 1);
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(y[4 * e]), "=r"(y[4 * e + 1]), "=r"(y[4 * e + 2]), "=r"(y[4 * e + 3])
                                 : "r"(v + row * 128 + (((piece ^ row) & 7) << 4)) : "memory");
                }
                pf_tmem_wait_ld();
                float odd = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) {                 // i >> 1: the tokens' eight, i & 1: the rows'
                    const int j = j0 + 8 * (i >> 1) + 2 * (lane & 3);
                    const float2 beta = *(const float2*)&dec.beta[j], upto = *(const float2*)&dec.upto[j];
                    const float z0 = beta.x * (__uint_as_float(y[i] << 16) - upto.x * __int_as_float(x[2 * i]));
                    const float z1 = beta.y * (__uint_as_float(y[i] & 0xffff0000u) - upto.y * __int_as_float(x[2 * i + 1]));
                    odd = fmaf(z0, 0.0f, fmaf(z1, 0.0f, odd));
                    x[2 * i] = __float_as_int(z0);
                    x[2 * i + 1] = __float_as_int(z1);
                }
                if (__builtin_expect(__any_sync(0xffffffffu, odd != 0.0f), 0))
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        float z = __int_as_float(x[i]);
                        clean(z, r16 * 16 + 8 * (i >> 1 & 1) + (lane >> 2), j0 + 8 * (i >> 2) + 2 * (lane & 3) + (i & 1));
                        x[i] = __float_as_int(z);
                    }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    f32x2 z = pk(__int_as_float(x[2 * i]), __int_as_float(x[2 * i + 1]));
                    w[0][i] = bf16_term(z);
                    w[1][i] = bf16_term(z);
                    w[2][i] = last_term(z);
                }
#pragma unroll
                for (int t = 0; t < 3; t++) tmem_st_16x4(tmem + kAtW + 32 * t + j0 / 2 + lanes + half, w[t]);
            }
            wait_st();
            pf_fence_before();
            __syncwarp();
            arrive_warp(&H.rhs_full);
            if (!wait_here(&H.x_full[k & 1], (k >> 1) & 1, &H)) { ok = false; break; }
            pf_fence_after();
#pragma unroll 1
            for (int r16 = 0; r16 < 2; r16++) {
                const uint32_t half = (uint32_t)(r16 * 16) << 16;
                int x[16];
                pf_tmem_ld_16x8<4>(tmem + kAtX + j0 + lanes + half, x);
                pf_tmem_wait_ld();
                float odd = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i++) odd = fmaf(__int_as_float(x[i]), 0.0f, odd);
                if (__builtin_expect(__any_sync(0xffffffffu, odd != 0.0f), 0))
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        float z = __int_as_float(x[i]);
                        clean(z, r16 * 16 + 8 * (i >> 1 & 1) + (lane >> 2), j0 + 8 * (i >> 2) + 2 * (lane & 3) + (i & 1));
                        x[i] = __float_as_int(z);
                    }
                uint32_t u[2][8], w[3][8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float2 left = *(const float2*)&dec.left[j0 + 8 * (i >> 1) + 2 * (lane & 3)];
                    f32x2 y = pk(__int_as_float(x[2 * i]), __int_as_float(x[2 * i + 1])), z = mul2(y, pk(left.x, left.y));
                    u[0][i] = bf16_term(y);
                    u[1][i] = last_term(y);
                    w[0][i] = bf16_term(z);
                    w[1][i] = bf16_term(z);
                    w[2][i] = last_term(z);
                }
#pragma unroll
                for (int t = 0; t < 2; t++) tmem_st_16x4(tmem + kAtSK + 32 * t + j0 / 2 + lanes + half, u[t]);
#pragma unroll
                for (int t = 0; t < 3; t++) tmem_st_16x4(tmem + kAtW + 32 * t + j0 / 2 + lanes + half, w[t]);
            }
            wait_st();
            pf_fence_before();
            __syncwarp();
            arrive_warp(&H.w_full);
            // (what the warp of the other half of the tokens has taken out of this one's rows comes with w_full)
            if (!wait_told_here(&H.u_full, k & 1, &H.w_full, k & 1, &H)) { ok = false; break; }
            pf_fence_after();
            const float by = dec.bad[row] >= C ? dec.whole : __int_as_float(0x7fffffff);     // (NaN: so becomes the row)
            const f32x2 by2 = pk(by, by);
#pragma unroll
            for (int e = 0; e < D / 2; e += 32) {
                int u[32];
                pf_tmem_ld32(tmem + kAtU + 64 * side + e + lanes, u);
                pf_tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const f32x2 x = fma2(by2, pk(s[e + i], s[e + i + 1]), pk(__int_as_float(u[i]), __int_as_float(u[i + 1])));
                    s[e + i] = lo_of(x);
                    s[e + i + 1] = hi_of(x);
                }
            }
            pf_fence_before();
        }
        if (ok && seq.to && !taken) store_state(s, seq.to + at, room, side * 16);            // (all that read the terms ended before the last U)
        if (!ok) give_up(SITE_CHAIN);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp < 12) {
            // ---- outputs
            uint8_t* out = c.out.data + (int64_t)seq.first * c.out.token + h * c.out.head + quarter * 64;
            for (int k = 0; k < chunks; k++, out += C * c.out.token) {
                const int n = min(C, seq.n - k * C);
                if (!wait_warp(&H.known[k % kRing], (k / kRing) & 1, &H) || !wait_warp(&H.w_full, k & 1, &H) || !wait_warp(&H.n_full, k & 1, &H)) {
                    give_up(SITE_OUT);
                    break;
                }
                pf_fence_after();
                const Decays& dec = H.ring[k % kRing];
                write_out(tmem + kAtR + lanes, tmem + kAtX + lanes, dec.upto, c.scale, [&](int r) { return dec.bad[quarter * 32 + r]; },
                          stages + (k % kStages) * kStage + kQK + quarter * 4096, out, c.out.token, n, &H.o_free);
                arrive_warp(&H.empty[k % kStages]);
            }
        } else if (warp < 14) {
            // ---- P: a token's row to a thread
            const int r = tid - 384;
            for (int k = 0; k < chunks; k++) {
                if (!wait_warp(&H.known[k % kRing], (k / kRing) & 1, &H) || !wait_warp(&H.qk_full[k & 1], (k >> 1) & 1, &H) ||
                    (k && !wait_warp(&H.n_full, (k - 1) & 1, &H))) {                 // the P before it has been read
                    give_up(SITE_P);
                    break;
                }
                pf_fence_after();
                weights_row(tmem + kAtQK + lanes, H.ring[k % kRing].log2, r, weights + r * 128, &H.qk_free);
                fence_async();
                __syncwarp();
                arrive_warp(&H.p_full);
            }
        } else if ((warp & 2) != 0) {
            // ---- T, by four warps that meet between the steps: the inverses of the four blocks of 16 on the diagonal by
            // substitution, then twice from two blocks and what is below the first of them
            //     [ A 0 ; L B ]^-1 = [ A^-1 0 ; -B^-1 L A^-1  B^-1 ]
            // (By substitution alone, a column to a thread, it took 17000 clocks a chunk, most of them the way to shared memory and
            // back.  The last two products by the warps' own matrix instructions and not by f32 ones, four rows of two columns to a thread: 232
            // to 228 us where a block has 32 chunks; L two columns to an instruction: to 224.)
            const int of = (warp & 1) | (warp >> 1 & 2);       // 0 to 3, of warps 18, 19, 14, 15
            float* const lower = (float*)(sm + (inverse + 3 * kP - pf_smem(sm)));       // L turned: [j][i]
            float* const between = lower + C * kL;                                      // 32 x 32, or two of 16 x 16
            float* const rows = (float*)(sm + (state + kTerm - pf_smem(sm)));           // T, in what the state's third term leaves
            float* const turned = rows + C * kT;                                        // [column][row within its 32]
            bool ok = wait_warp(&H.read, 0, &H);               // (the state on its way in has been there)
            for (int j = of * 32 + lane; j < C * (kT + kTurned) / 4; j += 128) *(float4*)(rows + 4 * j) = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int j = of * 32 + lane; j < 3 * 32 * 4; j += 128) {                    // and what is above T's blocks of 32 in its terms
                const int r = j >> 2 & 31;
                sts128(inverse + (j >> 7) * kP + r * 128 + (((4 + (j & 3)) ^ r) & 7) * 16, 0, 0, 0, 0);
            }
            for (int k = 0;; k++) {
                // They go on, or leave, together: nothing waits in a way that does not end but at these barriers, and a warp
                // comes to all of them.
                if (ok && k < chunks)
                    ok = wait_warp(&H.known[k % kRing], (k / kRing) & 1, &H) && wait_warp(&H.qk_full[k & 1], (k >> 1) & 1, &H);
                ok = all_of_four(ok);
                if (!ok || k == chunks) break;
                pf_fence_after();
                Decays& dec = H.ring[k % kRing];
                // row i of K K^T in lanes 64 + i: columns 0-15 and 16-31 of the first 32, 0-31 and 32-63 of the others
                const int i = (warp & 1) * 32 + lane, e0 = (warp >> 2 & 1) * (warp & 1 ? 32 : 16), e1 = e0 + (warp & 1 ? 32 : 16);
                const f32x2 g0 = pk(-dec.minus[0][i], -dec.minus[0][i]), g1 = pk(-dec.minus[1][i], -dec.minus[1][i]), beta2 = pk(dec.beta[i], dec.beta[i]);
                f32x2 odd2 = 0;
#pragma unroll 1
                for (int e = e0; e < e1; e += 16) {
                    int x[16];
                    pf_tmem_ld16(tmem + kAtQK + e + lanes, x);
                    pf_tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 z0 = *(const float4*)&dec.minus[0][e + j], z1 = *(const float4*)&dec.minus[1][e + j];
                        const f32x2 d[2] = {add2(add2(g0, pk(z0.x, z0.y)), add2(g1, pk(z1.x, z1.y))), add2(add2(g0, pk(z0.z, z0.w)), add2(g1, pk(z1.z, z1.w)))};
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            const int at = e + j + 2 * t;
                            const f32x2 y = mul2(mul2(beta2, pk(__int_as_float(x[j + 2 * t]), __int_as_float(x[j + 2 * t + 1]))),
                                                 pk(exp2_of(lo_of(d[t])), exp2_of(hi_of(d[t]))));
                            const f32x2 l = pk(at < i ? lo_of(y) : 0.0f, at + 1 < i ? hi_of(y) : 0.0f);
                            odd2 = fma2(l, 0, odd2);
                            lower[at * kL + i] = lo_of(l);
                            lower[(at + 1) * kL + i] = hi_of(l);
                        }
                    }
                }
                const float odd = lo_of(odd2) + hi_of(odd2);
                if (odd != 0.0f) {
                    // Something is not finite: rows of T from this one on will be NaN.  In the products it would meet the zeros of
                    // rows before it.
                    atomicMin(&dec.odd_row, i);
#pragma unroll 1
                    for (int j = e0; j < e1; j++)
                        if (!(fabsf(lower[j * kL + i]) <= 3.402823466e38f)) lower[j * kL + i] = 0.0f;
                }
                pf_fence_before();
                __syncwarp();
                arrive_warp(&H.qk_free);
                meet_four();
                // block `of` of 16: row r of a column is (r == column) - sum_{j < r} L_rj T_j, four rows at a time
                if (lane < 16) {
                    const float* own = lower + (16 * of) * kL + 16 * of;
                    float t[16];
#pragma unroll
                    for (int r0 = 0; r0 < 16; r0 += 4) {
#pragma unroll
                        for (int r = 0; r < 4; r++) t[r0 + r] = r0 + r == lane ? 1.0f : 0.0f;
#pragma unroll
                        for (int j = 0; j < r0 + 3; j++) {
                            const float4 l = *(const float4*)&own[j * kL + r0];
                            if (j < r0) t[r0] = fmaf(-l.x, t[j], t[r0]);
                            if (j < r0 + 1) t[r0 + 1] = fmaf(-l.y, t[j], t[r0 + 1]);
                            if (j < r0 + 2) t[r0 + 2] = fmaf(-l.z, t[j], t[r0 + 2]);
                            t[r0 + 3] = fmaf(-l.w, t[j], t[r0 + 3]);
                        }
                        *(float4*)&turned[(16 * of + lane) * kTurned + 16 * (of & 1) + r0] = make_float4(t[r0], t[r0 + 1], t[r0 + 2], t[r0 + 3]);
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++) rows[(16 * of + r) * kT + 16 * of + lane] = t[r];
                }
                meet_four();
                // the blocks of 32, two warps to each: four rows of a column to a thread
                const int b0 = 32 * (of >> 1), r4 = 8 * (of & 1) + 4 * (lane >> 4), c16 = lane & 15;
                float* const part = between + (of >> 1) * 256;
                float4 y = product4(lower + b0 * kL + b0 + 16 + r4, kL, rows + b0 * kT + b0 + c16, kT, 16);
                part[r4 * 16 + c16] = y.x; part[(r4 + 1) * 16 + c16] = y.y; part[(r4 + 2) * 16 + c16] = y.z; part[(r4 + 3) * 16 + c16] = y.w;
                meet_four();
                y = product4(turned + (b0 + 16) * kTurned + 16 + r4, kTurned, part + c16, 16, 16);
                float* to = rows + (b0 + 16 + r4) * kT + b0 + c16;
                to[0] = -y.x; to[kT] = -y.y; to[2 * kT] = -y.z; to[3 * kT] = -y.w;
                *(float4*)&turned[(b0 + c16) * kTurned + 16 + r4] = make_float4(-y.x, -y.y, -y.z, -y.w);
                meet_four();
                // and all of it: a tile of 16 x 16 to a warp
                const int m = 16 * (of >> 1), n = 16 * (of & 1);
                tile_product(lower + 32 + m, kL, rows + n, kT, between + m * kBetween + n, kBetween, 1.0f);
                meet_four();
                tile_product(turned + 32 * kTurned + m, kTurned, between + n, kBetween, rows + (32 + m) * kT + n, kT, -1.0f);
                meet_four();
                if (k && !wait_warp(&H.x_full[(k - 1) & 1], ((k - 1) >> 1) & 1, &H)) {           // the T before it has been read
                    ok = false;
                    continue;
                }
                // eight values of a row at a time as three bf16 terms, which are the values themselves
#pragma unroll 1
                for (int task = of * 32 + lane; task < 6 * C; task += 128) {
                    const int r = task < 128 ? task >> 2 : 32 + ((task - 128) >> 3), p = task < 128 ? task & 3 : task & 7;
                    const float4 a = *(const float4*)&rows[r * kT + 8 * p], b = *(const float4*)&rows[r * kT + 8 * p + 4];
                    f32x2 x[4] = {pk(a.x, a.y), pk(a.z, a.w), pk(b.x, b.y), pk(b.z, b.w)};
                    const uint32_t at = inverse + r * 128 + (((p ^ r) & 7) << 4), nan = r >= dec.odd_row ? 0x7fff7fffu : 0u;
#pragma unroll
                    for (int t = 0; t < 3; t++) {
                        uint32_t z[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) z[j] = (t < 2 ? bf16_term(x[j]) : last_term(x[j])) | nan;
                        sts128(at + t * kP, z[0], z[1], z[2], z[3]);
                    }
                }
                fence_async();
                __syncwarp();
                arrive_warp(&H.t_full);
            }
            if (!ok) give_up(SITE_T);
        } else if (warp == 16) {
            // ---- products
            if (pf_elect()) {
                bool ok = true;
                auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = ok && wait_one(bar, parity, &H); };
                auto stage = [&](int k) { return stages + (k % kStages) * kStage; };
                auto ready = [&] {
                    pf_fence_after();
                    fence_async();
                };
                auto qk_of = [&](int k) {
                    wait(&H.full[k % kStages], (k / kStages) & 1);
                    wait(&H.known[k % kRing], (k / kRing) & 1);      // (a chunk that is not full has been cleared)
                    if (k) wait(&H.qk_free, (k - 1) & 1);
                    if (!ok) return;
                    ready();
                    const uint64_t both = pf_desc_sw128(stage(k)), key = pf_desc_sw128(stage(k) + C * 128);
#pragma unroll 1
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            pf_mma_bf16(tmem + kAtQK, both + half * (kHalf >> 4) + 2 * e, key + half * (kHalf >> 4) + 2 * e, idesc(C, false, false), half || e);
                    pf_commit(&H.qk_full[k & 1]);
                };
                qk_of(0);
                for (int k = 0; k < chunks && ok; k++) {
                    wait(&H.s_full, k & 1);
                    if (k) wait(&H.o_free, (k - 1) & 1);
                    if (!ok) break;
                    ready();
                    // S [Q; K]^T, the third term for K alone: the outputs are rounded to bf16
                    const uint64_t third = pf_desc_sw128(state), both = pf_desc_sw128(stage(k)), key = pf_desc_sw128(stage(k) + C * 128);
#pragma unroll 1
                    for (int i = 0; i < 4; i++)              // of the first term, and of the second, the halves of dim_k
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            mma_ts(tmem + kAtR, tmem + kAtU + 64 * (i & 1) + 32 * (i >> 1) + 8 * e, both + (i & 1) * (kHalf >> 4) + 2 * e, idesc(2 * C, false, false), i || e);
#pragma unroll 1
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            pf_mma_bf16(tmem + kAtSK, third + half * (kHalf >> 4) + 2 * e, key + half * (kHalf >> 4) + 2 * e, idesc(C, false, false), 1);
                    pf_commit(&H.rk_full);
                    // The next chunk's Q K^T and K K^T, for its T: now, if its rows are here, else while u is made.
                    const int next = k + 1;
                    const bool more = next < chunks, now = more && pf_bar_try(&H.full[next % kStages], (next / kStages) & 1) &&
                                                            pf_bar_try(&H.known[next % kRing], (next / kRing) & 1) && pf_bar_try(&H.qk_free, k & 1);
                    if (now) qk_of(next);
                    wait(&H.rhs_full, k & 1);
                    wait(&H.t_full, k & 1);
                    if (!ok) break;
                    ready();
                    // T rhs by terms, the smallest products first: (T's, rhs's) = (0, 2) (1, 1) (2, 0) (1, 0) (0, 1) (0, 0)
                    const uint64_t t_at = pf_desc_sw128(inverse);
#pragma unroll 1
                    for (int i = 0; i < 6; i++) {
                        const uint32_t which = i == 0 ? 0 : i == 1 ? 1 : i == 2 ? 2 : i == 3 ? 1 : 0, of = i == 0 ? 2 : i == 1 || i == 4 ? 1 : 0;
#pragma unroll
                        for (int e = 0; e < C / 16; e++)
                            mma_ts(tmem + kAtX, tmem + kAtW + 32 * of + 8 * e, t_at + which * (kP >> 4) + 2 * e, idesc(C, false, false), i || e);
                    }
                    pf_commit(&H.x_full[k & 1]);
                    if (more && !now) qk_of(next);
                    wait(&H.w_full, k & 1);
                    if (!ok) break;
                    ready();
                    const uint64_t turned = desc_mn(stage(k) + C * 128, kHalf);
#pragma unroll 1
                    for (int i = 0; i < 3; i++)
#pragma unroll
                        for (int e = 0; e < C / 16; e++)
                            mma_ts(tmem + kAtU, tmem + kAtW + 32 * (2 - i) + 8 * e, turned + (2048 >> 4) * e, idesc(D, false, true), i || e);
                    pf_commit(&H.u_full);
                    pf_commit(&H.spent[k % kStages]);          // Q and K have been read
                    wait(&H.p_full, k & 1);
                    if (!ok) break;
                    ready();
                    const uint64_t weight = pf_desc_sw128(weights);
#pragma unroll
                    for (int e = 0; e < C / 8; e++)          // u's second term, then its first
                        mma_ts(tmem + kAtX, tmem + kAtSK + (e < 4 ? 32 : 0) + 8 * (e & 3), weight + 2 * (e & 3), idesc(C, false, false), e != 0);
                    pf_commit(&H.n_full);
                }
                if (!ok) {
                    atomicExch(c.status, SITE_MMA);
                    *(volatile int*)&H.abort = 1;
                }
            }
            __syncwarp();
            // nothing is in flight when the block ends, whatever ended the loop
            if (pf_elect()) pf_commit(&H.drained);
            __syncwarp();
            pf_bar_wait(&H.drained, 0);
            __syncwarp();
        } else if (warp == 17) {
            // ---- copies and decays: two tokens to a lane
            const int hq = h / c.group;
            int copies = 0, copies_v = 0;
            auto scalars_of = [&](int k, float (&g)[2], float (&beta)[2]) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int j = k * C + lane + 32 * i;
                    const bool here = j < seq.n;
                    g[i] = here ? c.decay[(int64_t)(seq.first + j) * c.decay_stride + h] : 0.0f;
                    beta[i] = here ? c.beta[(int64_t)(seq.first + j) * c.beta_stride + h] : 0.0f;
                }
            };
            float next_g[2], next_beta[2];
            scalars_of(0, next_g, next_beta);
            auto copy = [&](int k) {
                uint64_t* full = &H.full[k % kStages];
                const uint32_t at = stages + (k % kStages) * kStage;
                const int token = seq.first + k * C;
                copies++;
                if (lane == 0) {
                    pf_bar_expect_tx(full, 4 * C * 128);
                    for (int half = 0; half < 2; half++) {
                        box(at + half * kHalf, &maps.q, half * 64, hq, token, full);
                        box(at + half * kHalf + C * 128, &maps.k, half * 64, hq, token, full);
                    }
                }
                __syncwarp();
            };
            auto copy_v = [&](int k) {
                uint64_t* full = &H.full_v[k % kStages];
                const uint32_t at = stages + (k % kStages) * kStage + kQK;
                copies_v++;
                if (lane == 0) {
                    pf_bar_expect_tx(full, 2 * C * 128);
                    for (int half = 0; half < 2; half++) box(at + half * (C * 128), &maps.v, half * 64, h, seq.first + k * C, full);
                }
                __syncwarp();
            };
            // Q and K of a stage are free when its products are done, V's place when its outputs have been by way of it.
            auto v_may = [&](int k) { return wait_warp(&H.empty[k % kStages], ((k / kStages) & 1) ^ 1, &H); };
            for (int k = 0; k < kStages && k < chunks; k++) {
                copy(k);
                copy_v(k);
            }
            for (int k = 0; k < chunks; k++) {
                const int n = min(C, seq.n - k * C);
                // the copies before the decays, whose next ones are on their way meanwhile
                if (k >= kStages) {
                    if (!wait_warp(&H.spent[k % kStages], ((k / kStages) & 1) ^ 1, &H)) { give_up(SITE_COPY); break; }
                    copy(k);
                }
                const float g[2] = {clamp_decay(next_g[0]), clamp_decay(next_g[1])}, beta[2] = {next_beta[0], next_beta[1]};
                scalars_of(k + 1, next_g, next_beta);
                double x[2];
                const double whole = sums_of_decays(g, x);
                Decays& dec = H.ring[k % kRing];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int j = lane + 32 * i;
                    const double y = x[i] * 1.4426950408889634;
                    dec.log2[j] = (float)y;
                    dec.minus[0][j] = -(float)y;
                    dec.minus[1][j] = (float)((double)(float)y - y);
                    dec.left[j] = j < n ? expf((float)(whole - x[i])) : 0.0f;
                    dec.upto[j] = expf((float)x[i]);
                    dec.beta[j] = beta[i];
                }
#pragma unroll
                for (int i = 0; i < 4; i++) dec.bad[lane + 32 * i] = C;
                if (lane == 0) {
                    dec.whole = expf((float)whole);
                    dec.odd_row = C;
                }
                if (n < C) {                                   // the last: its V before it is told
                    if (k >= kStages) {
                        if (!v_may(k)) { give_up(SITE_COPY); break; }
                        copy_v(k);
                    }
                    if (!wait_warp(&H.full[k % kStages], (k / kStages) & 1, &H) || !wait_warp(&H.full_v[k % kStages], (k / kStages) & 1, &H)) {
                        give_up(SITE_COPY);
                        break;
                    }
                    clear_rows(stages + (k % kStages) * kStage, n);
                }
                __syncwarp();
                arrive_warp(&H.known[k % kRing]);
                if (n == C && k >= kStages) {
                    if (!v_may(k)) { give_up(SITE_COPY); break; }
                    copy_v(k);
                }
            }
            // no copy is under way when the block ends, whatever ended the loop
            if (copies) wait_for_last_fills<kStages, 1>((uint32_t)(copies - 1), (uint32_t)copies, [&](uint32_t slot, uint32_t parity) { pf_bar_wait(&H.full[slot], parity); });
            if (copies_v) wait_for_last_fills<kStages, 1>((uint32_t)(copies_v - 1), (uint32_t)copies_v, [&](uint32_t slot, uint32_t parity) { pf_bar_wait(&H.full_v[slot], parity); });
            __syncwarp();
        }
    }
    pf_fence_before();
    __syncthreads();
    pf_fence_after();
    if (warp == 16) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

int g_regs = 0;                                      // a thread's, as built

}  // namespace

cudaError_t linear_delta_attributes() {
    cudaFuncAttributes f;
    cudaError_t e = cudaFuncGetAttributes(&f, linear_delta_kernel);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(linear_delta_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess) g_regs = f.numRegs;
    return e;
}

bool launch_linear_delta(const LinearCall& c, cudaStream_t stream, cudaError_t* e) {
    // setmaxnreg deals out the registers that the block was launched with: a build that launches with fewer would wait for ever
    if (g_regs * kThreads < kChain * kChainRegs + (kThreads - kChain) * kOtherRegs) return false;
    Maps maps;
    if (!map_rows(&maps.q, c.q, c.n_head / c.group, c.n_tokens) || !map_rows(&maps.k, c.k, c.n_head / c.group, c.n_tokens) ||
        !map_rows(&maps.v, c.v, c.n_head, c.n_tokens))
        return false;
    count_launch();
    *e = launch_with(false, stream, linear_delta_kernel, dim3((unsigned)(c.n_seq * c.n_head)), dim3(kThreads), (size_t)kSmem, c, maps);
    return true;
}

}  // namespace bivmoe
