// Linear attention token by token: the recurrent form, for single tokens and drafts, and for every type and
// dimension that the kernels for prompts do not take, with or without the delta rule.
//
// A row of the state S [dim_v][dim_k] evolves by itself: row r needs v[r], the token's k and q, and nothing
// of the other rows.  So the rows of all heads and requests are shared out over the chip, a warp holding
// 4 R of them in registers (eight lanes to a row, four neighbouring values of dim_k each), and no row is
// read or written more than once however many tokens there are.  For a token
//     o = scale (a (S q) + u (q k)),   u = v   or, with beta,   u = beta (v - a (S k)),   S = a S + u k
// where S is the state before it: both products meet the old state, so one round of shuffles joins them,
// and the update is not on the way to the output.  Arithmetic is f32, two values to an instruction.
//
// Single tokens are bound by the states' way from memory and back (64 requests x 32 heads of 128 x 128: 268 MB in 46 us, 0.89 of the
// measured rate), drafts by the products as well, long requests by the way of a token through its products and shuffles: 530
// clocks, 2048 tokens of 32 heads in 555 us.
#include "common.cuh"
#include "launch.cuh"
#include "linear.cuh"
#include "tcgen05.cuh"

namespace bivmoe {

namespace {

constexpr int kThreads = 128, kWarps = 4;

// TB: tokens whose rows are brought in together.  (1: single tokens, without the code for more.)
template <int DK, int R, int TB> struct Steps {
    static constexpr int rows = kWarps * 4 * R;      // of dim_v, to a thread block
    static constexpr int raw = (2 * DK + rows) * 4;  // bytes of a token's k, q and v, as f32 at most
    struct Shared {
        uint8_t in[2][TB][raw];
        float k[TB][DK], q[TB][DK], v[TB][rows], o[TB][rows];
        float a[TB], rest[TB], b[TB], qk[TB];
    };
};

__device__ __forceinline__ void copy16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// Eight lanes' values joined, in every one of them.
__device__ __forceinline__ float join8(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    return x + __shfl_xor_sync(0xffffffffu, x, 4);
}
// N values of a type, from shared memory, as f32
template <int N> __device__ __forceinline__ void widen(const uint8_t* from, int ty, int at, float (&x)[N]) {
    if (ty == BIVMOE_F32) {
#pragma unroll
        for (int i = 0; i < N; i += 2) *(float2*)&x[i] = *(const float2*)(from + (at + i) * 4);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const uint32_t w = *(const uint32_t*)(from + (at + i) * 2);
        if (ty == BIVMOE_BF16) {
            x[i] = __uint_as_float(w << 16);
            x[i + 1] = __uint_as_float(w & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*(const __half2*)&w);
            x[i] = f.x;
            x[i + 1] = f.y;
        }
    }
}

template <int DK, int R, int TB, bool DELTA>
__global__ void __launch_bounds__(kThreads, DK == 256 ? 3 : TB == 1 ? 5 : 4) linear_steps_kernel(const __grid_constant__ LinearCall c) {
    using P = Steps<DK, R, TB>;
    constexpr bool kLong = TB == 16;
    constexpr int N4 = DK / 32, PER = DK / 32;       // pieces of four values of a lane in a row; a lane's values of a row of q or k
    extern __shared__ __align__(16) uint8_t smem[];
    auto& sh = *(typename P::Shared*)smem;
    pdl_enter();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane >> 3, part = lane & 7;
    const int slices = c.dim_v / P::rows, h = blockIdx.x / slices, row0 = (blockIdx.x % slices) * P::rows, b = blockIdx.y;
    const LinearSeq seq = linear_seq(c, b);
    const bool mine = slot_taken(c, b, tid, kThreads);
    if (!seq.n) return;
    const int ty = c.type, es = type_size(ty), per = 16 / es;
    const int nq = DK / per, nv = P::rows / per, nv_shift = 31 - __clz(nv);      // 16-byte pieces of a token's k or q, and of its v
    const int hq = h / c.group;
    const uint8_t *kp = c.k.data + hq * c.k.head, *qp = c.q.data ? c.q.data + hq * c.q.head : nullptr,
                  *vp = c.v.data + h * c.v.head + (int64_t)row0 * es;
    const int k_bytes = DK * es;

    // a block of tokens' rows, asked for: a warp to a token's k and q
    auto bring = [&](int block) {
        const int t0 = block * TB, n = min(TB, seq.n - t0);
        for (int t = warp; t < n; t += kWarps) {
            const int64_t row = seq.first + t0 + t;
            uint8_t* to = sh.in[block & 1][t];
            for (int p = lane; p < nq; p += 32) {
                copy16(to + p * 16, kp + row * c.k.token + p * 16);
                if (qp) copy16(to + k_bytes + p * 16, qp + row * c.q.token + p * 16);
            }
        }
        for (int i = tid; i < n << nv_shift; i += kThreads) {
            const int t = i >> nv_shift, p = i & (nv - 1);
            copy16(sh.in[block & 1][t] + 2 * k_bytes + p * 16, vp + (int64_t)(seq.first + t0 + t) * c.v.token + p * 16);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // and its decays and betas, a token to a thread
    float next_a = 0.0f, next_b = 0.0f;
    auto scalars = [&](int block) {
        const int t = block * TB + tid;
        if (tid < TB && t < seq.n) {
            const int64_t row = seq.first + t;
            next_a = c.decay[row * c.decay_stride + h];
            if (DELTA) next_b = c.beta[row * c.beta_stride + h];
        }
    };
    bring(0);
    scalars(0);

    f32x2 s[R][2 * N4];
    const int64_t at = (int64_t)h * c.head + (int64_t)(row0 + warp * 4 * R + sub) * DK + part * 4;    // row r of a lane: 4 r further on
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int i = 0; i < N4; i++) {
            const float4 x = seq.from ? __ldcs((const float4*)(seq.from + at + r * 4 * DK + i * 32)) : make_float4(0.f, 0.f, 0.f, 0.f);
            s[r][2 * i] = pk(x.x, x.y);
            s[r][2 * i + 1] = pk(x.z, x.w);
        }
    const bool taken = __syncthreads_or(mine);
    if (taken)
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < 2 * N4; i++) s[r][i] = 0;

    auto keep = [&] {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < N4; i++)
                __stcs((float4*)(seq.to + at + r * 4 * DK + i * 32),
                       make_float4(lo_of(s[r][2 * i]), hi_of(s[r][2 * i]), lo_of(s[r][2 * i + 1]), hi_of(s[r][2 * i + 1])));
    };
    const int blocks = (seq.n + TB - 1) / TB;
    for (int block = 0; block < blocks; block++) {
        const int t0 = block * TB, n = min(TB, seq.n - t0);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();                             // the rows are here; the last block's outputs and k, q, v are done with
        const uint8_t* in = sh.in[block & 1][0];
        for (int t = warp; t < n; t += kWarps) {
            float k[PER], q[PER], qk = 0.0f;
            widen<PER>(in + t * P::raw, ty, lane * PER, k);
#pragma unroll
            for (int i = 0; i < PER; i += 2) *(float2*)&sh.k[t][lane * PER + i] = *(const float2*)&k[i];
            if (qp) {
                widen<PER>(in + t * P::raw + k_bytes, ty, lane * PER, q);
#pragma unroll
                for (int i = 0; i < PER; i += 2) *(float2*)&sh.q[t][lane * PER + i] = *(const float2*)&q[i];
#pragma unroll
                for (int i = 0; i < PER; i++) qk = fmaf(k[i], q[i], qk);
                qk = join8(qk);
                qk += __shfl_xor_sync(0xffffffffu, qk, 8);
                qk += __shfl_xor_sync(0xffffffffu, qk, 16);
                if (lane == 0) sh.qk[t] = qk;
            }
        }
        for (int i = tid; i < n << nv_shift; i += kThreads) {
            const int t = i >> nv_shift, p = i & (nv - 1);
            widen16(*(const uint4*)(in + t * P::raw + 2 * k_bytes + p * 16), ty, sh.v[t] + p * per);
        }
        if (tid < TB) {
            // Over many tokens the decay's own rounding would be most of what the state loses: what f32 leaves of it goes along.
            if constexpr (kLong) {
                const double a = exp((double)clamp_decay(next_a));
                sh.a[tid] = (float)a;
                sh.rest[tid] = (float)(a - (double)(float)a);
            } else {
                sh.a[tid] = expf(clamp_decay(next_a));
            }
            if (DELTA) sh.b[tid] = next_b;
        }
        bring(block + 1);
        scalars(block + 1);
        __syncthreads();
        // Tokens from..to, without a branch between one and the next: their loads, products and shuffles overlap, and only the
        // state's update (with the delta rule: the way to u, too) is a chain.
        auto tokens = [&](int from, int to) {
#pragma unroll TB == 1 ? 1 : TB == 8 && DK > 64 ? 2 : 4
            for (int t = from; t < to; t++) {
                const float a = sh.a[t], beta = DELTA ? sh.b[t] : 1.0f, qk = sh.qk[t];
                const float rest = kLong ? sh.rest[t] : 0.0f;
                const f32x2 a2 = pk(a, a), rest2 = pk(rest, rest);
                f32x2 k2[2 * N4], ks[R][2] = {}, qs[R][2] = {};
#pragma unroll
                for (int i = 0; i < N4; i++) {
                    const float4 x = *(const float4*)(sh.k[t] + part * 4 + i * 32);
                    k2[2 * i] = pk(x.x, x.y);
                    k2[2 * i + 1] = pk(x.z, x.w);
                    if (DELTA)
#pragma unroll
                        for (int r = 0; r < R; r++)
#pragma unroll
                            for (int e = 0; e < 2; e++) ks[r][e] = fma2(s[r][2 * i + e], k2[2 * i + e], ks[r][e]);
                }
#pragma unroll
                for (int i = 0; i < N4; i++) {
                    const float4 x = *(const float4*)(sh.q[t] + part * 4 + i * 32);
                    const f32x2 q2[2] = {pk(x.x, x.y), pk(x.z, x.w)};
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int e = 0; e < 2; e++) qs[r][e] = fma2(s[r][2 * i + e], q2[e], qs[r][e]);
                }
                auto sum = [](const f32x2 (&x)[2]) {
                    const f32x2 y = add2(x[0], x[1]);
                    return lo_of(y) + hi_of(y);
                };
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const int row = warp * 4 * R + r * 4 + sub;
                    float u = sh.v[t][row];
                    if (DELTA) u = beta * (u - a * join8(sum(ks[r])));
                    const f32x2 u2 = pk(u, u);
#pragma unroll
                    for (int i = 0; i < 2 * N4; i++) {
                        const f32x2 x = mul2(u2, k2[i]);
                        s[r][i] = fma2(a2, s[r][i], kLong ? fma2(rest2, s[r][i], x) : x);
                    }
                    const float o = c.scale * fmaf(a, join8(sum(qs[r])), u * qk);
                    if (part == 0) sh.o[t][row] = o;
                }
            }
        };
        const int kept = min(max(seq.kept - t0, 0), n);
        if (seq.to && !taken && kept > 0 && seq.kept <= t0 + n) {
            tokens(0, kept);
            keep();
            tokens(kept, n);
        } else {
            tokens(0, n);
        }
        if (qp) {
            __syncthreads();
            uint8_t* op = c.out.data + h * c.out.head + (int64_t)row0 * es;
            for (int i = tid; i < n << nv_shift; i += kThreads) {
                const int t = i >> nv_shift, p = i & (nv - 1);
                *(uint4*)(op + (int64_t)(seq.first + t0 + t) * c.out.token + p * 16) = narrow16(sh.o[t] + p * per, ty);
            }
        }
    }
}

template <int DK, int R, int TB> cudaError_t set_attributes() {
    const int bytes = sizeof(typename Steps<DK, R, TB>::Shared);
    cudaError_t e = cudaFuncSetAttribute(linear_steps_kernel<DK, R, TB, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return e == cudaSuccess ? cudaFuncSetAttribute(linear_steps_kernel<DK, R, TB, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) : e;
}
template <int DK, int R, int TB> cudaError_t launch(const LinearCall& c, cudaStream_t stream) {
    count_launch();
    const dim3 grid(c.n_head * (c.dim_v / Steps<DK, R, TB>::rows), c.n_seq);
    const size_t smem = sizeof(typename Steps<DK, R, TB>::Shared);
    // Scheduled early, except where long requests' blocks would all run at once: those would be put where the kernel before leaves room, several
    // to one multiprocessor, and stay there.  (One request of 2048 tokens, 32 heads of f32, calls one after another: early 697 to 839 us, else 554; with
    // the delta rule 888 to 1099 and 672; 12 tokens 9.5 and 8.4.  Of more blocks, 8 requests of 9 tokens 19.8 and 20.8, 64 of 16 184 and 186, 16 of
    // 512 and heads of 64 362 and 365; drafts of few blocks, one request of 5, 4.7 and 6.9, single tokens of two 4.8 and 6.1.)
    const bool early = TB < 16 || (int64_t)grid.x * grid.y >= 4 * c.sms;
    return launch_with(pdl_mode() == 1 || (pdl_mode() != 0 && early), stream, c.beta ? linear_steps_kernel<DK, R, TB, true> : linear_steps_kernel<DK, R, TB, false>, grid,
                       dim3(kThreads), smem, c);
}
// Rows to a thread, and tokens brought in together.  us with one, two, four rows: 64 single tokens, 32 heads of 128: 59, 46, 47; 128 of 16
// heads of 64: 32, 18, 15; 32 of 16 heads of 256: 64, 49, -; 32 requests of 5 tokens, delta rule, 65, 42, 38.  Long requests, eight
// tokens together and sixteen: one of 2048, 32 heads, f32: 737 and 619, 690 and 555, 999 and 741; 16 of 512, 32 heads of 64: 584 and 527, 401 and
// 363, 342 and 327 (one of 2048, 16 heads, sixteen tokens: 442, 481, 587); one of 2048, 16 heads of 256, delta rule: 1172 and 1028, 1139 and 988 (4
// heads: 777, 985; eight of 500 by 16 heads: 1750, 1222).  The loop with two tokens in hand (four for prompts and heads of 64; one for single tokens) took 37.0 us for the 32 drafts, with
// one 41.9, with four 37.7; the single tokens with four 48.3 and not 46.
// (Prompts before what f32 leaves of a decay went along, which takes a tenth: 507 to 555 us; nine requests of up to 1224 tokens, f32, delta
// rule, were off by 1.1e-6 without it and are by 2.5e-7.)
template <int DK> cudaError_t launch_rows(const LinearCall& c, int max_new, int sm_count, cudaStream_t stream) {
    constexpr int single = DK == 64 ? 4 : 2, drafts = DK == 256 ? 2 : 4, prompts = DK == 256 ? 1 : 2;
    const int64_t rows = (int64_t)c.n_seq * c.n_head * c.dim_v;
    const bool many = rows >= (int64_t)sm_count * 256, some = rows >= (int64_t)sm_count * 64;
    if (max_new == 1) return many ? launch<DK, single, 1>(c, stream) : some ? launch<DK, 2, 1>(c, stream) : launch<DK, 1, 1>(c, stream);
    if (max_new > 8) return launch<DK, prompts, 16>(c, stream);
    return many ? launch<DK, drafts, 8>(c, stream) : some ? launch<DK, 2, 8>(c, stream) : launch<DK, 1, 8>(c, stream);
}
template <int DK> cudaError_t all_attributes() {
    constexpr int single = DK == 64 ? 4 : 2, drafts = DK == 256 ? 2 : 4, prompts = DK == 256 ? 1 : 2;
    for (cudaError_t e : {set_attributes<DK, single, 1>(), set_attributes<DK, 2, 1>(), set_attributes<DK, 1, 1>(), set_attributes<DK, drafts, 8>(),
                          set_attributes<DK, 2, 8>(), set_attributes<DK, 1, 8>(), set_attributes<DK, prompts, 16>()})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}

}  // namespace

cudaError_t linear_attributes() {
    for (cudaError_t e : {all_attributes<64>(), all_attributes<128>(), all_attributes<256>()})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}

cudaError_t launch_linear_steps(const LinearCall& c, int max_new, int sm_count, cudaStream_t stream) {
    switch (c.dim_k) {
        case 64: return launch_rows<64>(c, max_new, sm_count, stream);
        case 128: return launch_rows<128>(c, max_new, sm_count, stream);
        default: return launch_rows<256>(c, max_new, sm_count, stream);
    }
}

}  // namespace bivmoe
