// Linear attention on the fifth-generation tensor cores: what its kernels share.  Products of 128 rows of bf16 with f32 sums, waits
// that end, rows by the copy engine.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <limits.h>

#include "cache.cuh"
#include "linear.cuh"
#include "tcgen05.cuh"

namespace bivmoe {

namespace {

constexpr int C = 64, D = 128;                       // tokens of a chunk, values of a head
constexpr int kHalf = 128 * 128;                     // 64 values of a chunk's Q rows, then its K rows: 128 bytes each
constexpr int kQK = 2 * kHalf, kV = 2 * C * 128;

// The request that a block takes: the longest first, so that the last blocks to set out are short.  (Requests of 1 to 3000 tokens, 9 x 32
// heads, 131 -> 107 us; with the delta rule, 1 to 1500, 256 -> 220, before its other steps.)  Every warp finds it by itself; of more than 64 requests
// the blocks are many, and their order matters little, as it does where all blocks run at once.
__device__ __forceinline__ int request_at(const LinearCall& c, int at) {
    if (c.n_seq > 64 || c.n_seq < 2 || (int)gridDim.x <= c.sms) return at;
    const int lane = threadIdx.x & 31;
    int n[2], rank[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; i++) n[i] = lane + 32 * i < c.n_seq ? rows_of(c.first[lane + 32 * i], c.first[lane + 32 * i + 1], c.n_tokens).n : INT_MIN;
    const int any = __shfl_sync(0xffffffffu, n[0], 0);
    if (__all_sync(0xffffffffu, (n[0] == any || n[0] == INT_MIN) && (n[1] == any || n[1] == INT_MIN))) return at;
    for (int j = 0; j < c.n_seq; j++) {
        const int m = __shfl_sync(0xffffffffu, j < 32 ? n[0] : n[1], j & 31);
#pragma unroll
        for (int i = 0; i < 2; i++) rank[i] += m > n[i] || (m == n[i] && j < lane + 32 * i);
    }
    const unsigned low = __ballot_sync(0xffffffffu, lane < c.n_seq && rank[0] == at);
    const unsigned high = __ballot_sync(0xffffffffu, lane + 32 < c.n_seq && rank[1] == at);
    return low ? __ffs(low) - 1 : 31 + __ffs(high);
}

// What every wait of a block looks at: H has an int `abort`.
template <class H> __device__ __forceinline__ uint64_t look_here(const H* h, uint32_t turn, uint64_t t0) {      // where the clock began; 0: gives up
    WaitClock clock{t0};
    if (*(const volatile int*)&h->abort) return 0;
    return clock.late(turn, pf_now_ns(), false) ? 0 : clock.t0;
}
template <class H> __device__ __noinline__ uint64_t look(const H* h, uint32_t turn, uint64_t t0) { return look_here(h, turn, t0); }
// HERE: no call in it.  A call keeps few registers, and a state that lives across one was stored and loaded for it in every turn
// of the loop, whether or not it was made.
template <class H, bool CLUSTER, bool HERE> struct Wait {
    uint64_t* bar;
    uint32_t parity;
    const H* h;
    uint64_t t0 = 0;
    __device__ __forceinline__ bool ready() const {
        if (!CLUSTER) return pf_bar_try(bar, parity);
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(pf_smem(bar)), "r"(parity) : "memory");
        return ok != 0;
    }
    __device__ __forceinline__ bool late(uint32_t turn) { return !(t0 = HERE ? look_here(h, turn, t0) : look(h, turn, t0)); }
    __device__ __forceinline__ void pause() const {}
    __device__ __forceinline__ bool all(bool v) const { return __all_sync(0xffffffffu, v); }
};
// A product's end, and behind it the word of the warp whose writes are read then (not by way of the issuing thread, which tells the
// product's end).  It has long been given, and both are asked for in one turn, so that it costs no trip of its own.
template <class H, bool HERE> struct WaitTold : Wait<H, false, HERE> {
    uint64_t* word;
    uint32_t word_parity;
    __device__ __forceinline__ WaitTold(uint64_t* bar, uint32_t parity, uint64_t* word, uint32_t word_parity, const H* h)
        : Wait<H, false, HERE>{bar, parity, h}, word(word), word_parity(word_parity) {}
    __device__ __forceinline__ bool ready() const {
        const bool ended = pf_bar_try(this->bar, this->parity), told = pf_bar_try(word, word_parity);      // (in this order)
        return ended && told;
    }
};
template <class H> __device__ __forceinline__ bool wait_told(uint64_t* bar, uint32_t parity, uint64_t* word, uint32_t word_parity, const H* h) {
    return bounded_wait_together<64>(WaitTold<H, false>{bar, parity, word, word_parity, h});
}
template <class H> __device__ __forceinline__ bool wait_told_here(uint64_t* bar, uint32_t parity, uint64_t* word, uint32_t word_parity, const H* h) {
    return bounded_wait_together<64>(WaitTold<H, true>{bar, parity, word, word_parity, h});
}
template <class H> __device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, const H* h) {
    return bounded_wait<64>(Wait<H, false, false>{bar, parity, h});
}
template <class H> __device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, const H* h) {
    return bounded_wait_together<64>(Wait<H, false, false>{bar, parity, h});
}
template <bool CLUSTER = false, class H> __device__ __forceinline__ bool wait_here(uint64_t* bar, uint32_t parity, const H* h) {
    return bounded_wait_together<64>(Wait<H, CLUSTER, true>{bar, parity, h});
}
__device__ __forceinline__ void arrive_warp(uint64_t* bar) {
    if ((threadIdx.x & 31) == 0) pf_bar_arrive(bar);
    __syncwarp();
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 16 lanes x 16 columns of this warp's 32 lanes (`at`: the first of the 16): register 2 j + i of lane l is lane l / 4 + 8 i, column
// 4 j + l % 4
__device__ __forceinline__ void tmem_st_16x4(uint32_t at, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
    return v;
}
// A (128 rows) in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// bf16, f32 sums, 128 rows; A or B along its rows (MN-major) instead of along K
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// MN-major, 128-byte swizzle: 64 values are a row of 128 bytes, eight rows an atom of 1024; `next` bytes on to the next 64 values
__device__ __forceinline__ uint64_t desc_mn(uint32_t at, uint32_t next) {
    return (uint64_t)((at & 0x3FFFFu) >> 4) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// The first copy by a map waits for the map itself, 2600 clocks and more: asked for while a block sets out.
__device__ __forceinline__ void prefetch_maps(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c) {
    for (const CUtensorMap* m : {&a, &b, &c}) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}
__device__ __forceinline__ void box(uint32_t dst, const CUtensorMap* map, int value, int head, int token, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(value), "r"(head), "r"(token), "r"(pf_smem(bar)) : "memory");
}

// A warp's 32 rows of a state, 512 bytes each, between memory and the threads' registers: by way of 16 KB of shared memory of the
// warp's own, so that memory is met in whole rows.  Piece p of row r stands at p ^ r (of eight).  (By its own row's pieces, from each
// thread, a state took 5 us each way.)
__device__ __forceinline__ uint32_t state_piece(uint32_t room, int r, int p) { return room + r * 512 + ((p & ~7) << 4) + (((p ^ r) & 7) << 4); }
// (P pieces of each row, from p0 on: a warp may have a part of the rows' length)
template <int P> __device__ __forceinline__ void ask_for_state(const float* from, uint32_t room, int p0) {
    const int lane = threadIdx.x & 31;
#pragma unroll 8
    for (int i = 0; i < P; i++) {
        const int r = (i * 32 + lane) / P, p = p0 + (i * 32 + lane) % P;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(state_piece(room, r, p)), "l"(from + r * D + p * 4) : "memory");
    }
}
// (of what this warp has asked for)
__device__ __forceinline__ void wait_for_state() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
}
template <int N> __device__ __forceinline__ void store_state(const float (&s)[N], float* to, uint32_t room, int p0) {
    constexpr int P = N / 4;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int p = 0; p < P; p++)
        sts128(state_piece(room, lane, p0 + p), __float_as_uint(s[4 * p]), __float_as_uint(s[4 * p + 1]), __float_as_uint(s[4 * p + 2]), __float_as_uint(s[4 * p + 3]));
    __syncwarp();
#pragma unroll
    for (int i0 = 0; i0 < P; i0 += 8) {
        uint4 w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = lds128(state_piece(room, ((i0 + i) * 32 + lane) / P, p0 + ((i0 + i) * 32 + lane) % P));
#pragma unroll
        for (int i = 0; i < 8; i++) *(uint4*)(to + ((i0 + i) * 32 + lane) / P * D + (p0 + ((i0 + i) * 32 + lane) % P) * 4) = w[i];
    }
}

// P = Q K^T and its decays of a token (a row of tensor memory, in its own thread), rounded to bf16, in a row of 128 bytes of shared
// memory (128-byte swizzle).  After its last load from tensor memory the warp arrives at `free`.  The exponent is a difference of sums in
// f32, of up to 64 x 128 log2(e) (tokens whose decays are all at the end of their range): off by 2^-10 then, and the weight by 7e-4 of
// itself, where bf16 rounds it by up to 2^-9; sums of some hundreds, as decays have them in earnest, by 2^-16.
__device__ __forceinline__ void weights_row(uint32_t from, const float* log2, int r, uint32_t row, uint64_t* free) {
    const float g = log2[r];
#pragma unroll 1
    for (int e = 0; e < C; e += 16) {
        int x[16];
        pf_tmem_ld16(from + e, x);
        float l[16];
#pragma unroll
        for (int i = 0; i < 16; i += 4) *(float4*)(l + i) = *(const float4*)&log2[e + i];
        pf_tmem_wait_ld();
        if (e + 16 == C) {
            pf_fence_before();
            __syncwarp();
            arrive_warp(free);
        }
        uint32_t p[8];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            float y[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                y[t] = __int_as_float(x[i + t]) * exp2_of(g - l[i + t]);
                if (e + i + t > r) y[t] = 0.0f;
            }
            p[i / 2] = narrow2(y[0], y[1], BIVMOE_BF16);
        }
        sts128(row + (((e / 8 ^ r) & 7) << 4), p[0], p[1], p[2], p[3]);
        sts128(row + (((e / 8 + 1 ^ r) & 7) << 4), p[4], p[5], p[6], p[7]);
    }
}

// A warp's 32 values of a chunk's outputs, scale (upto R + N), by way of 4 KB of shared memory, so that they are written in pieces of
// 16 bytes (two bytes at a time, from the lanes they stand in, held everything up for 4300 clocks a chunk).  bad(r): the first
// token from which row r is NaN.  After its last load from tensor memory the warp arrives at `free`.
template <class Bad>
__device__ __forceinline__ void write_out(uint32_t r_at, uint32_t n_at, const float* upto, float scale, Bad bad, uint32_t tile, uint8_t* out, int64_t token,
                                          int n, uint64_t* free) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int part = 0; part < 4; part++) {                     // 16 values of 32 tokens
        const int r0 = (part >> 1) * 16, i0 = (part & 1) * 32;
        int x[16], y[16];
        pf_tmem_ld_16x8<4>(r_at + i0 + ((uint32_t)r0 << 16), x);
        pf_tmem_ld_16x8<4>(n_at + i0 + ((uint32_t)r0 << 16), y);
        const int first[2] = {bad(r0 + (lane >> 2)), bad(r0 + 8 + (lane >> 2))};
        const bool any = __any_sync(0xffffffffu, min(first[0], first[1]) < C);
        pf_tmem_wait_ld();
        if (part == 3) {
            pf_fence_before();
            __syncwarp();
            arrive_warp(free);
        }
        uint32_t o[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = i0 + 8 * e + 2 * (lane & 3);
            const float2 by = *(const float2*)&upto[i];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                float u = scale * fmaf(by.x, __int_as_float(x[4 * e + 2 * t]), __int_as_float(y[4 * e + 2 * t]));
                float v = scale * fmaf(by.y, __int_as_float(x[4 * e + 2 * t + 1]), __int_as_float(y[4 * e + 2 * t + 1]));
                if (any) {
                    if (i >= first[t]) u = __int_as_float(0x7fffffff);
                    if (i + 1 >= first[t]) v = __int_as_float(0x7fffffff);
                }
                o[2 * e + t] = narrow2(u, v, BIVMOE_BF16);
            }
        }
        // eight tokens' rows of eight values, turned: rows of 64 bytes, piece p of row r at p ^ (r / 2)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int row = i0 + 16 * e + 8 * (lane >> 4) + (lane & 7), p = (part >> 1) * 2 + (lane >> 3 & 1);
            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(tile + row * 64 + ((p ^ (row >> 1 & 3)) << 4)),
                         "r"(o[4 * e]), "r"(o[4 * e + 1]), "r"(o[4 * e + 2]), "r"(o[4 * e + 3]) : "memory");
        }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int row = 8 * i + (lane >> 2), p = lane & 3;
        const uint4 w = lds128(tile + row * 64 + ((p ^ (row >> 1 & 3)) << 4));
        if (row < n) *(uint4*)(out + (int64_t)row * token + p * 16) = w;
    }
    fence_async();
    __syncwarp();
}

// The first of the three bf16 terms that make two f32 values, by cutting off; what is left of them.
__device__ __forceinline__ uint32_t bf16_term(f32x2& x) {
    const uint32_t a = (uint32_t)x, b = (uint32_t)(x >> 32);
    x = fma2((f32x2)(a & 0xffff0000u) | (f32x2)(b & 0xffff0000u) << 32, pk(-1.0f, -1.0f), x);
    return __byte_perm(a, b, 0x7632);
}
// the last of them, which is all that is left
__device__ __forceinline__ uint32_t last_term(f32x2 x) { return __byte_perm((uint32_t)x, (uint32_t)(x >> 32), 0x7632); }
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                 "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
// Sums of a chunk's decays up to each token, two to a lane (tokens lane and lane + 32); returns the whole.
__device__ __forceinline__ double sums_of_decays(const float (&g)[2], double (&x)[2]) {
    const int lane = threadIdx.x & 31;
    x[0] = g[0];
    x[1] = g[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const double y = __shfl_up_sync(0xffffffffu, x[i], o);
            if (lane >= o) x[i] += y;
        }
    x[1] += __shfl_sync(0xffffffffu, x[0], 31);
    return __shfl_sync(0xffffffffu, x[1], 31);
}

// A chunk of n tokens: the rows of K and V behind them are another request's: zeros, so that nothing of them reaches a sum.
__device__ __forceinline__ void clear_rows(uint32_t stage, int n) {
    const int lane = threadIdx.x & 31;
    for (int i = lane; i < (C - n) * 32; i += 32) {
        const int row = n + (i >> 5), p = i & 31;              // 16-byte pieces: K's 16, V's 16
        const uint32_t to = p < 16 ? stage + (p >> 3) * kHalf + C * 128 : stage + kQK + ((p >> 3) & 1) * (C * 128);
        sts128(to + row * 128 + (p & 7) * 16, 0, 0, 0, 0);
    }
    fence_async();
}

// rows [token][head][128] as boxes of 64 tokens x 64 values
bool map_rows(CUtensorMap* m, const LinearRows& r, int heads, int64_t tokens) {
    static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess) cudaGetLastError();
        return (PFN_cuTensorMapEncodeTiled_v12000)(found == cudaDriverEntryPointSuccess ? f : nullptr);
    }();
    if (!encode) return false;
    const int64_t head = heads > 1 ? r.head : D * 2, token = tokens > 1 ? r.token : heads * head;
    if (head <= 0 || token <= 0) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)head, (cuuint64_t)token};
    const cuuint32_t part[3] = {64, 1, C}, step[3] = {1, 1, 1};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, r.data, dims, strides, part, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

}  // namespace bivmoe
