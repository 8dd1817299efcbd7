// Linear attention with a decay for each head: what its kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/bivmoe.h"
#include "rows_of.h"

namespace bivmoe {

constexpr int kLinearSeqs = 1024;    // requests of a call

struct LinearRows {
    uint8_t* data;
    int64_t token, head;             // strides in bytes
};
// The arguments as the kernels take them.
struct LinearCall {
    LinearRows q, k, v, out;         // q.data null: no outputs
    const float *decay, *beta;
    int64_t decay_stride, beta_stride;
    float* states;
    int64_t slot, head, n_slots;     // strides in values
    const int32_t *slots, *first, *past, *keep;
    int32_t* status;
    int n_seq, n_tokens, n_head, group, dim_k, dim_v, type, sms;
    float scale;
};

// A request of a call: its rows, where its state is read and written from, after how many tokens.
struct LinearSeq {
    int first, n, kept;
    float *from, *to;                // the state of a head is at + head * c.head; null: zeros, not kept
};
// One thread's part in finding out whether an earlier request has the slot already (of `threads` threads; the block
// has to combine the answers): of two requests with one slot the first alone has it, whatever order blocks run in.
__device__ __forceinline__ bool slot_taken(const LinearCall& c, int b, int thread, int threads) {
    const int slot = c.slots[b];
    bool taken = false;
    for (int i = thread; i < b; i += threads) taken |= c.slots[i] == slot;
    return taken;
}
__device__ __forceinline__ LinearSeq linear_seq(const LinearCall& c, int b) {
    LinearSeq s;
    const RowsOf rows = rows_of(c.first[b], c.first[b + 1], c.n_tokens);
    s.first = rows.first;
    s.n = rows.n;
    s.kept = c.keep ? min(max(c.keep[b], 0), s.n) : s.n;
    const int slot = c.slots[b];
    float* at = slot >= 0 && slot < c.n_slots ? c.states + slot * c.slot : nullptr;
    s.from = c.past && c.past[b] == 0 ? nullptr : at;
    s.to = s.kept > 0 ? at : nullptr;
    return s;
}

// Above zero counts as zero; below -128 the exponential is zero in f32 in any case, and a sum of
// decays with -infinity or a type's lowest value in it would lose the ones beside it.  NaN stays.
__device__ __forceinline__ float clamp_decay(float g) { return g > 0.0f ? 0.0f : g < -128.0f ? -128.0f : g; }

__host__ __device__ constexpr int type_size(int ty) { return ty == BIVMOE_F32 ? 4 : 2; }

// 16 bytes of a type as f32
__device__ __forceinline__ void widen16(const uint4& raw, int ty, float* to) {
    if (ty == BIVMOE_F32) {
        *(uint4*)to = raw;
        return;
    }
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float2 f;
        if (ty == BIVMOE_BF16) f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        else f = __half22float2(*(const __half2*)&w[i]);
        *(float2*)(to + 2 * i) = f;
    }
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, int ty) {
    if (ty == BIVMOE_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *(const uint32_t*)&h;
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
}
// as many f32 values as 16 bytes of a type hold, rounded once
__device__ __forceinline__ uint4 narrow16(const float* f, int ty) {
    if (ty == BIVMOE_F32) return *(const uint4*)f;
    return make_uint4(narrow2(f[0], f[1], ty), narrow2(f[2], f[3], ty), narrow2(f[4], f[5], ty), narrow2(f[6], f[7], ty));
}

cudaError_t linear_attributes();     // once for each device, before a capture
cudaError_t linear_chunks_attributes();
// bf16 rows, heads of 128 x 128, outputs, no delta rule, the state kept after all tokens; false where the rows' strides are
// none that the copy engine takes
cudaError_t linear_delta_attributes();
bool launch_linear_delta(const LinearCall& c, cudaStream_t stream, cudaError_t* e);   // the same with the delta rule
bool launch_linear_chunks(const LinearCall& c, int max_new, cudaStream_t stream, cudaError_t* e);
cudaError_t launch_linear_steps(const LinearCall& c, int max_new, int sm_count, cudaStream_t stream);

}  // namespace bivmoe
