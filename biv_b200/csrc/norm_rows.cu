// Root-mean-square norm of rows, with the residual's addition, a silu gate, and rows of floats or of 8 bits with
// scales: one pass over memory.
//
// Bytes bound it.  A row's threads keep its values in registers between the sum and the product, eight
// neighbouring values to a thread and step; rows of up to 32 pieces' threads stay within a warp, wider ones
// have a thread block.  The squares are summed in f64: with that the order of the sum does not reach the
// root once it is rounded to f32, so that y, and with y the codes of 8-bit rows, are the same however many
// threads share a row (a code flips at a border of its rounding, 1/127 of the block's largest value, when y
// is off by one bit).  It costs one conversion and one f64 product a value, of which an SM does 16 a clock:
// 4.5 T a second against the 1.6 T that the memory brings at the smallest rows of 2 + 2 bytes a value.
#include <cuda_fp8.h>

#include <type_traits>

#include "cache.cuh"
#include "common.cuh"
#include "launch.cuh"
#include "norm.cuh"

namespace bivmoe {

namespace {

__device__ __forceinline__ uint32_t pack2(float a, float b, int ty) {
    if (ty == BIVMOE_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *(const uint32_t*)&h;
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
}
// Eight values as they lie in memory
template <int TY> struct Piece {
    uint4 raw[TY == BIVMOE_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
        for (int i = 0; i < (TY == BIVMOE_F32 ? 2 : 1); i++) raw[i] = *(const uint4*)(p + 16 * i);
    }
    __device__ __forceinline__ void store(uint8_t* p) const {
#pragma unroll
        for (int i = 0; i < (TY == BIVMOE_F32 ? 2 : 1); i++) *(uint4*)(p + 16 * i) = raw[i];
    }
    __device__ __forceinline__ void round(const float (&v)[8]) {
        if constexpr (TY == BIVMOE_F32) {
            raw[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            raw[TY == BIVMOE_F32] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
        } else {
            raw[0] = make_uint4(pack2(v[0], v[1], TY), pack2(v[2], v[3], TY), pack2(v[4], v[5], TY), pack2(v[6], v[7], TY));
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        if constexpr (TY == BIVMOE_F32) {
            const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __uint_as_float(w[i]);
            return;
        }
        const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (TY == BIVMOE_BF16) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*(const __half2*)&w[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
};
template <int TY> __device__ __forceinline__ void load8_of(const uint8_t* p, float (&v)[8]) {
    Piece<TY> x;
    x.load(p);
    x.values(v);
}
__device__ __forceinline__ void store8(uint8_t* p, int ty, const float (&v)[8]) {
    if (ty == BIVMOE_F32) {
        *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)(p + 16) = make_float4(v[4], v[5], v[6], v[7]);
        return;
    }
    *(uint4*)p = make_uint4(pack2(v[0], v[1], ty), pack2(v[2], v[3], ty), pack2(v[4], v[5], ty), pack2(v[6], v[7], ty));
}
__device__ __forceinline__ float load1(const uint8_t* p, int ty) {
    return ty == BIVMOE_F32 ? *(const float*)p : ty == BIVMOE_BF16 ? __bfloat162float(*(const __nv_bfloat16*)p) : __half2float(*(const __half*)p);
}
__device__ __forceinline__ void store1(uint8_t* p, int ty, float v) {
    if (ty == BIVMOE_F32) *(float*)p = v;
    else if (ty == BIVMOE_BF16) *(__nv_bfloat16*)p = __float2bfloat16_rn(v);
    else *(__half*)p = __float2half_rn(v);
}
__device__ __forceinline__ float rounded(float v, int ty) {
    return ty == BIVMOE_F32 ? v : ty == BIVMOE_BF16 ? __bfloat162float(__float2bfloat16_rn(v)) : __half2float(__float2half_rn(v));
}
// z / (1 + exp(-z)).  exp(-z) = 2^t (1 + r ln 2), t the f32 product with -log2(e) and r what that leaves (the product's own
// rounding, and that of the constant): 2^-22 of it wrong at most, as the reciprocal's is.  From z = -87 down the result is zero.  (With expf and a
// division, rounded to half a step, 262144 rows of 128 bf16 values took 65 us and not 62, before the other steps; two values to an
// instruction 41.0 and not 41.6.)
__device__ __forceinline__ float silu(float z) {
    constexpr float log2e = 1.44269504f, rest = 1.92596303e-8f, ln2 = 0.693147181f;        // log2(e) = log2e + rest
    const float t = __fmul_rn(z, -log2e), r = __fmaf_rn(z, -rest, __fmaf_rn(z, -log2e, -t));
    float e, i;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    if (fabsf(t) < 126.0f) e = __fmaf_rn(__fmul_rn(e, ln2), r, e);       // (elsewhere e is 0, infinity, or NaN, and r may be NaN)
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(i) : "f"(__fadd_rn(1.0f, e)));
    return __fmul_rn(z, i);
}
// 1 / sqrt(mean + eps), rounded once to f32.  From an f32 estimate, 2^-22 off, by a step of third order: 2^-64 of it are left, less than f64's
// own rounding.  (A root and a division in f64, a hundred operations for each thread of a row.)
__device__ __forceinline__ float root_of(double sum, const NormCall& c) {
    const double s = sum * c.per_value + c.eps;
    if (!(s > 1e-30 && s < 1e30)) return (float)(1.0 / sqrt(s));         // (what f32 may not hold; NaN)
    const double y = (double)rsqrtf((float)s), e = fma(-s * y, y, 1.0);
    return (float)fma(y * e, fma(0.375, e, 0.5), y);
}
// The eight codes of y in Q8: halves away from zero, for |q| < 2^23: what is below one half stays below it when the largest number below one
// half is added, and a half reaches the next whole number by rounding; what is behind the point falls off as 2^23 is added.  (A
// conversion to an integer is one for 16 lanes a clock.)  A scale of few bits, among f32's smallest numbers, may be rounded by up to half of
// itself, so that quotients pass 127 (2^-149 for a largest value of 190 of it): they stay at 127, which elsewhere none passes, the scale being off
// by 2^-24 of itself at most.
__device__ __forceinline__ uint2 q8_codes(const float (&y)[8], float scale) {
    const float inv = scale != 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    float q[8];
    if (isinf(inv)) {                                // f32 does not hold it
#pragma unroll 1
        for (int j = 0; j < 8; j++) {
            float x = y[0];
#pragma unroll
            for (int i = 1; i < 8; i++) x = i == j ? y[i] : x;
            x = __fdiv_rn(x, scale);
            x = x > 127.0f ? 127.0f : x < -127.0f ? -127.0f : x;
#pragma unroll
            for (int i = 0; i < 8; i++) q[i] = i == j ? x : q[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = __fmul_rn(y[j], inv);
    }
    uint32_t n[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t whole = __float_as_uint(__fadd_rz(fabsf(q[j]) + 0.49999997f, 8388608.0f)), sign = (uint32_t)(__float_as_int(q[j]) >> 31);
        n[j] = (whole ^ sign) - sign;
    }
    auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410); };
    return make_uint2(four(n[0], n[1], n[2], n[3]), four(n[4], n[5], n[6], n[7]));
}
// y / scale, rounded to f32, as E4M3: from the product with the reciprocal by a step on the remainder, which leaves the quotient rounded
// as a division rounds it (Markstein, 1990).  What a scale near f32's ends does not allow is divided.  (The division for every
// value: 16384 rows of 4096 bf16 108 us, with this 70.)
struct ByScale {
    float scale, inv;
    __device__ __forceinline__ float of(float y) const {
        if (inv == 0.0f) return scale != 0.0f ? __fdiv_rn(y, scale) : 0.0f;
        const float q = __fmul_rn(y, inv);
        return __fmaf_rn(__fmaf_rn(-q, scale, y), inv, q);
    }
    __device__ __forceinline__ uint32_t e4m3(float y) const { return (uint32_t)__nv_cvt_float_to_fp8(of(y), __NV_SATFINITE, __NV_E4M3); }
    __device__ __forceinline__ uint2 e4m3(const float (&y)[8]) const {
        uint32_t two[4];
        if (inv == 0.0f) {
#pragma unroll 1
            for (int j = 0; j < 4; j++) {
                const float a = j & 2 ? j & 1 ? y[6] : y[4] : j & 1 ? y[2] : y[0], b = j & 2 ? j & 1 ? y[7] : y[5] : j & 1 ? y[3] : y[1];
                const uint32_t x = e4m3(a) | e4m3(b) << 8;
#pragma unroll
                for (int i = 0; i < 4; i++) two[i] = i == j ? x : two[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float q[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    q[i] = __fmul_rn(y[2 * j + i], inv);
                    q[i] = __fmaf_rn(__fmaf_rn(-q[i], scale, y[2 * j + i]), inv, q[i]);
                }
                two[j] = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
            }
        }
        return make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
    }
};
__device__ __forceinline__ ByScale by_scale(float s) { return {s, s > 1e-25f && s < 1e37f ? __fdiv_rn(1.0f, s) : 0.0f}; }
// The larger of two magnitudes, by their bits, or NaN where one is: its bits are above infinity's.
__device__ __forceinline__ float top(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }

// Sum (f64) or maximum over the threads of a row: `tpr` of them, a part of a warp or the thread block.
template <class T, class F> __device__ __forceinline__ T join(T x, int tpr, T* room, F f) {
    const int in_warp = min(tpr, 32);
    for (int o = in_warp >> 1; o; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
    if (tpr > 32) {
        if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = x;
        __syncthreads();
        x = room[0];
        for (int i = 1; i < tpr >> 5; i++) x = f(x, room[i]);
    }
    return x;
}

// K pieces of eight values of a row in a thread's registers, as they lie in memory, and a gate of 16 bits, too, so that it is under way
// while the squares are summed; rows of 16 bits take 64 registers a thread, for twice the warps.  The kernel is short of
// instructions before it is short of bytes, where rows are of 16 bits: so nothing branches between the loads and the stores.
// (262144 rows of 128 bf16, gated, 201 MB: 41 us, 4.9 TB/s; with f32 values in the registers, the gate asked for after the sum,
// and branches around the places behind a row, 62.  16384 rows of 4096 bf16 with add, 537 MB: 81 us, 6.6 TB/s; with add's type looked at
// piece by piece, 108.  16381 rows of 2048 f32 with add to Q8, 440 MB: 70 us, 6.3 TB/s.)
template <int K, int XT, int KIND, bool GATED>
__global__ void __launch_bounds__(K == 4 ? 512 : 1024, K == 4 && XT != BIVMOE_F32 ? 2 : 1) norm_rows_kernel(const __grid_constant__ NormCall c, int tpr) {
    __shared__ double room[32];
    __shared__ float room_top[32];
    pdl_enter();
    constexpr int XS = XT == BIVMOE_F32 ? 4 : 2;
    const int shift = 31 - __clz(tpr), in = threadIdx.x & (tpr - 1);       // (tpr is a power of two)
    const int64_t r = (int64_t)blockIdx.x * (blockDim.x >> shift) + (threadIdx.x >> shift);
    const bool here = r < c.rows;
    const uint32_t row = here ? (uint32_t)r : 0;
    const int64_t token = c.heads.div(row);
    const int head = row - (int)token * c.heads.d;
    uint8_t* x = c.x.data + token * c.x.token + head * c.x.head;
    const uint8_t* add = c.add.data ? c.add.data + token * c.add.token + head * c.add.head : nullptr;
    const uint8_t* gate = c.gate.data + token * c.gate.token + head * c.gate.head;
    const bool ahead = GATED && c.gate.size == 2;
    auto mine = [&](int k) { return here && (in + k * tpr) * 8 < c.width; };
    // Places behind the row are zeros, and go through the arithmetic as the others do: only loads and stores ask.
    Piece<XT> v[K];
    uint4 g[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        v[k] = Piece<XT>{};
        if (mine(k)) v[k].load(x + (in + k * tpr) * 8 * XS);
    }
    if (add) {
        // all loads before the first store, which the compiler may not move them over, and before the first use
        auto join_with = [&](auto type) {
            constexpr int AT = decltype(type)::value;
            Piece<AT> w[K];
#pragma unroll
            for (int k = 0; k < K; k++)
                if (mine(k)) w[k].load(add + (in + k * tpr) * 8 * (AT == BIVMOE_F32 ? 4 : 2));
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (!mine(k)) continue;
                float f[8], g[8];
                v[k].values(f);
                w[k].values(g);
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] += g[j];
                v[k].round(f);
                v[k].store(x + (in + k * tpr) * 8 * XS);
            }
        };
        if (c.add.type == BIVMOE_F32) join_with(std::integral_constant<int, BIVMOE_F32>());
        else if (c.add.type == BIVMOE_BF16) join_with(std::integral_constant<int, BIVMOE_BF16>());
        else join_with(std::integral_constant<int, BIVMOE_F16>());
    }
    if (GATED)
#pragma unroll
        for (int k = 0; k < K; k++) {
            g[k] = make_uint4(0, 0, 0, 0);
            if (ahead && mine(k)) g[k] = *(const uint4*)(gate + (in + k * tpr) * 16);
        }
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < K; k++) {
        float f[8];
        v[k].values(f);
#pragma unroll
        for (int j = 0; j < 8; j++) sum = fma((double)f[j], (double)f[j], sum);
    }
    sum = join(sum, tpr, room, [](double a, double b) { return a + b; });
    const float root = root_of(sum, c);
    uint8_t* out = c.out.data + token * c.out.token + head * c.out.head;
    float most = 0.0f, kept[KIND == BIVMOE_NORM_E4M3 ? K : 1][8];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int i = (in + k * tpr) * 8;
        float y[8], w[8];
        v[k].values(y);
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = 1.0f;
        if (c.weight) load8_of<BIVMOE_F32>((const uint8_t*)(c.weight + (mine(k) ? i : 0)), w);
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = __fmul_rn(__fmul_rn(y[j], root), w[j]);
        if (GATED) {
            if (!ahead) {
                if (mine(k)) load8_of<BIVMOE_F32>(gate + i * 4, w);
            } else if (c.gate.type == BIVMOE_BF16) {
                Piece<BIVMOE_BF16>{g[k]}.values(w);
            } else {
                Piece<BIVMOE_F16>{g[k]}.values(w);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = __fmul_rn(y[j], silu(w[j]));
        }
        if constexpr (KIND == 0) {
            if (mine(k)) store8(out + i * c.out.size, c.out.type, y);
            continue;
        }
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) m = top(m, fabsf(y[j]));
        if (!mine(k)) m = 0.0f;
        if (KIND == BIVMOE_NORM_E4M3 && c.block == 0) {      // the row's scale: when all of it is there
            most = top(most, m);
#pragma unroll
            for (int j = 0; j < 8; j++) kept[KIND == BIVMOE_NORM_E4M3 ? k : 0][j] = y[j];
            continue;
        }
        const int block = KIND == BIVMOE_NORM_Q8 ? 32 : 128;
#pragma unroll
        for (int o = 1; o < block / 8; o <<= 1) m = top(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float scale = __fmul_rn(m, KIND == BIVMOE_NORM_Q8 ? 1.0f / 127.0f : 1.0f / 448.0f);
        uint2 code;
        if constexpr (KIND == BIVMOE_NORM_Q8) {
            code = q8_codes(y, scale);
        } else {
            code = by_scale(scale).e4m3(y);
        }
        if (mine(k)) {
            *(uint2*)(out + i) = code;
            if (i % block == 0) c.scales[token * c.scales_stride + head * (c.width / block) + i / block] = scale;
        }
    }
    if (KIND != BIVMOE_NORM_E4M3 || c.block != 0) return;
    most = join(most, tpr, room_top, [](float a, float b) { return top(a, b); });
    const float scale = __fmul_rn(most, 1.0f / 448.0f);
    const ByScale by = by_scale(scale);
#pragma unroll
    for (int k = 0; k < K; k++) {
        if (!mine(k)) continue;
        *(uint2*)(out + (in + k * tpr) * 8) = by.e4m3(kept[KIND == BIVMOE_NORM_E4M3 ? k : 0]);
    }
    if (here && in == 0) c.scales[token * c.scales_stride + head] = scale;
}

// Rows of any width, alignment and length, value by value: read again for each step.  A thread meets the same
// places in each, so that what it wrote to x, or reads of an x that is also the output, is its own.
__global__ void __launch_bounds__(256) norm_any_kernel(const NormCall c) {
    __shared__ double room[32];
    __shared__ float room_top[32];
    pdl_enter();
    const uint32_t row = blockIdx.x;
    const int64_t token = c.heads.div(row);
    const int head = row - (int)token * c.heads.d, tpr = blockDim.x;
    uint8_t* x = c.x.data + token * c.x.token + head * c.x.head;
    const uint8_t* add = c.add.data ? c.add.data + token * c.add.token + head * c.add.head : nullptr;
    const uint8_t* gate = c.gate.data ? c.gate.data + token * c.gate.token + head * c.gate.head : nullptr;
    uint8_t* out = c.out.data + token * c.out.token + head * c.out.head;
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < c.width; i += tpr) {
        float v = load1(x + i * c.x.size, c.x.type);
        if (add) {
            v = rounded(v + load1(add + i * c.add.size, c.add.type), c.x.type);
            store1(x + i * c.x.size, c.x.type, v);
        }
        sum = fma((double)v, (double)v, sum);
    }
    sum = join(sum, tpr, room, [](double a, double b) { return a + b; });
    const float root = root_of(sum, c);
    auto value = [&](int64_t i) {
        float y = __fmul_rn(__fmul_rn(load1(x + i * c.x.size, c.x.type), root), c.weight ? c.weight[i] : 1.0f);
        return gate ? __fmul_rn(y, silu(load1(gate + i * c.gate.size, c.gate.type))) : y;
    };
    if (c.kind == 0) {
        for (int64_t i = threadIdx.x; i < c.width; i += tpr) store1(out + i * c.out.size, c.out.type, value(i));
        return;
    }
    // 8-bit rows come here with a scale for the row alone
    float most = 0.0f;
    for (int64_t i = threadIdx.x; i < c.width; i += tpr) most = top(most, fabsf(value(i)));
    most = join(most, tpr, room_top, [](float a, float b) { return top(a, b); });
    const float scale = __fmul_rn(most, 1.0f / 448.0f);
    const ByScale by = by_scale(scale);
    for (int64_t i = threadIdx.x; i < c.width; i += tpr) out[i] = (uint8_t)by.e4m3(value(i));
    if (threadIdx.x == 0) c.scales[token * c.scales_stride + head] = scale;
}

template <int K, int XT, bool GATED> cudaError_t launch_of(const NormCall& c, int tpr, cudaStream_t stream) {
    const int threads = tpr > 32 ? tpr : 128, rows = threads / tpr;
    auto* kernel = c.kind == 0 ? norm_rows_kernel<K, XT, 0, GATED> : c.kind == BIVMOE_NORM_Q8 ? norm_rows_kernel<K, XT, BIVMOE_NORM_Q8, GATED>
                                                                                               : norm_rows_kernel<K, XT, BIVMOE_NORM_E4M3, GATED>;
    return launch_with(pdl_mode() != 0, stream, kernel, dim3((unsigned)((c.rows + rows - 1) / rows)), dim3(threads), 0, c, tpr);
}
template <int K, int XT> cudaError_t launch_of(const NormCall& c, int tpr, cudaStream_t stream) {
    return c.gate.data ? launch_of<K, XT, true>(c, tpr, stream) : launch_of<K, XT, false>(c, tpr, stream);
}
template <int K> cudaError_t launch(const NormCall& c, int tpr, cudaStream_t stream) {
    return c.x.type == BIVMOE_F32 ? launch_of<K, BIVMOE_F32>(c, tpr, stream)
         : c.x.type == BIVMOE_BF16 ? launch_of<K, BIVMOE_BF16>(c, tpr, stream) : launch_of<K, BIVMOE_F16>(c, tpr, stream);
}

}  // namespace

// In registers where rows, strides and width allow pieces of eight values (`vector`).  A thread block for a row of
// 512 threads x 4 pieces holds 16384 values.
bool norm_fits(int width, bool vector) { return vector && width % 8 == 0 && width <= 16384; }

cudaError_t launch_norm(const NormCall& c, bool vector, int sm_count, cudaStream_t stream) {
    count_launch();
    if (!norm_fits(c.width, vector)) {
        int threads = 32;
        while (threads < 256 && threads * 4 < c.width) threads *= 2;
        return launch_with(pdl_mode() != 0, stream, norm_any_kernel, dim3((unsigned)c.rows), dim3(threads), 0, c);
    }
    const int pieces = c.width / 8, least = c.block ? c.block / 8 : 1;
    int tpr = 1;
    while (tpr < pieces || tpr < least) tpr *= 2;
    // Many rows: four pieces to a thread, for more bytes under way, and because the root, in f64, costs a warp as much as some
    // tens of pieces.
    if (tpr > 1024 || (c.rows * tpr >= sm_count * 4096 && tpr >= 4 * least && tpr > 4)) return launch<4>(c, tpr / 4, stream);
    return launch<1>(c, tpr, stream);
}

}  // namespace bivmoe
