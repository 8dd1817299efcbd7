// The C ABI of what stands beside the cache: linear attention's handles and calls, the norm, the verification.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <new>

#include "common.cuh"
#include "linear.cuh"
#include "norm.cuh"
#include "verify.cuh"

using namespace bivmoe;

struct bivmoe_linear {
    bivmoe_linear_desc d{};
    int sm_count = 0;
    int32_t* status = nullptr;       // device: a bounded wait gave up
};

static int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return global_error(code, buf);
}
static int cuda_fail(cudaError_t e, const char* what) {
    return fail(e == cudaErrorMemoryAllocation ? BIVMOE_ERR_OOM : BIVMOE_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
static bool aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }
static bool is_float(int ty) { return ty == BIVMOE_F32 || ty == BIVMOE_F16 || ty == BIVMOE_BF16; }

// Rows that are written: a stride of zero (a broadcast tensor's) would put one over another.
static bool over_one_another(const bivmoe_rows& r, int tokens, int heads) { return (tokens > 1 && !r.stride_token) || (heads > 1 && !r.stride_head); }

// The multiprocessors of a device that this library has code for; asked for once a device.
static int device_of(int device, const char* what, int* sms) {
    static std::atomic<int> known[64];
    if (device >= 0 && device < 64 && (*sms = known[device].load(std::memory_order_relaxed)) > 0) return BIVMOE_OK;
    int major = 0, n = 0;
    cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return cuda_fail(e, what);
    if (major != 10)
        return fail(BIVMOE_ERR_UNSUPPORTED, "device %d is of compute capability %d.x; this library is built for sm_100a only", device, major);
    if (device < 64) known[device].store(n, std::memory_order_relaxed);
    *sms = n;
    return BIVMOE_OK;
}

// ---- linear attention ----

// New tokens of a request up to which they are taken one by one.  (us of 32 heads of 128, one by one and by the kernels for prompts: one
// request of 24 tokens 10.4 and 11.9; 16 of 16 39 and 39, of 24 58 and 39; 64 of 16 150 and 140, of 24 225 and 141.  With the delta rule: 12.4 and
// 16.5; 48 and 59, 72 and 59; 183 and 203, 273 and 203.)
constexpr int kSteps = 16;

extern "C" void bivmoe_linear_destroy(bivmoe_linear* l) {
    if (!l) return;
    DeviceScope on_device(l->d.device);
    if (l->status) cudaFree(l->status);
    delete l;
}

extern "C" int bivmoe_linear_create(const bivmoe_linear_desc* d, bivmoe_linear** out) {
    if (out) *out = nullptr;
    if (!d || !out) return fail(BIVMOE_ERR_ARGUMENT, "null descriptor or output");
    if (!is_float(d->ggml_type)) return fail(BIVMOE_ERR_UNSUPPORTED, "rows of type %d: F32, F16 and BF16 have kernels", d->ggml_type);
    for (int dim : {d->dim_k, d->dim_v})
        if (dim != 64 && dim != 128 && dim != 256)
            return fail(BIVMOE_ERR_UNSUPPORTED, "dim_k %d, dim_v %d: 64, 128 and 256 have kernels", d->dim_k, d->dim_v);
    if (d->n_head_qk < 1 || d->n_head < 1 || d->n_head > 1024 || d->n_head % d->n_head_qk)
        return fail(BIVMOE_ERR_ARGUMENT, "n_head %d (at most 1024) is not a multiple of n_head_qk %d", d->n_head, d->n_head_qk);
    if (d->max_seqs < 1 || d->max_seqs > kLinearSeqs) return fail(BIVMOE_ERR_ARGUMENT, "max_seqs %d outside 1..%d", d->max_seqs, kLinearSeqs);
    DeviceScope on_device(d->device);
    int cur = -1, sms = 0;
    cudaError_t e = cudaGetDevice(&cur);
    if (e == cudaSuccess && cur != d->device) e = cudaSetDevice(d->device);   // reports an invalid ordinal
    if (e != cudaSuccess) return cuda_fail(e, "bivmoe_linear_create");
    if (int rc = device_of(d->device, "bivmoe_linear_create", &sms)) return rc;
    bivmoe_linear* l = new (std::nothrow) bivmoe_linear();
    if (!l) return fail(BIVMOE_ERR_OOM, "host allocation failed");
    l->d = *d;
    l->sm_count = sms;
    e = linear_attributes();
    if (e == cudaSuccess) e = linear_chunks_attributes();
    if (e == cudaSuccess) e = linear_delta_attributes();
    if (e == cudaSuccess) e = dev_alloc((void**)&l->status, 16);
    if (e == cudaSuccess) e = cudaMemset(l->status, 0, 16);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();   // the clear, before a call on any stream
    if (e != cudaSuccess) {
        const int rc = cuda_fail(e, "bivmoe_linear_create");
        bivmoe_linear_destroy(l);
        return rc;
    }
    *out = l;
    return BIVMOE_OK;
}

extern "C" int bivmoe_linear_attend(bivmoe_linear* l, const bivmoe_linear_args* a, void* stream) {
    if (!l || !a) return fail(BIVMOE_ERR_ARGUMENT, "null layer or arguments");
    const bivmoe_linear_desc& d = l->d;
    if (a->n_seq < 0 || a->n_seq > d.max_seqs) return fail(BIVMOE_ERR_ARGUMENT, "n_seq = %d outside 0..max_seqs = %d", a->n_seq, d.max_seqs);
    if (a->n_tokens < 0) return fail(BIVMOE_ERR_ARGUMENT, "n_tokens = %d", a->n_tokens);
    if (a->max_new < 0) return fail(BIVMOE_ERR_ARGUMENT, "max_new = %d", a->max_new);
    if (!a->n_seq || !a->n_tokens) return BIVMOE_OK;
    const int per = 16 / type_size(d.ggml_type);
    const struct { const char* name; const bivmoe_rows* r; bool may_lack; } rows[] = {
        {"q", &a->q, true}, {"k", &a->k, false}, {"v", &a->v, false}, {"out", &a->out, !a->q.data}};
    for (const auto& x : rows) {
        if (!x.r->data && x.may_lack) continue;
        if (!x.r->data) return fail(BIVMOE_ERR_ARGUMENT, "%s: null pointer", x.name);
        if (x.r->ggml_type != d.ggml_type) return fail(BIVMOE_ERR_ARGUMENT, "%s: not of the layer's type", x.name);
        if (!aligned(x.r->data, 16) || x.r->stride_token % per || x.r->stride_head % per)
            return fail(BIVMOE_ERR_ARGUMENT, "%s: not aligned to 16 bytes, or a stride is not a multiple of them", x.name);
    }
    if (a->q.data && over_one_another(a->out, a->n_tokens, d.n_head)) return fail(BIVMOE_ERR_ARGUMENT, "out: rows lie over one another");
    // q and k are read by the blocks of all heads that share them, v by those alone that write its place of out, and before they do
    if (a->q.data && (a->out.data == a->q.data || a->out.data == a->k.data ||
                      (a->out.data == a->v.data && ((a->n_tokens > 1 && a->out.stride_token != a->v.stride_token) ||
                                                    (d.n_head > 1 && a->out.stride_head != a->v.stride_head)))))
        return fail(BIVMOE_ERR_ARGUMENT, "out may be v, with its strides, but not q or k");
    if (!a->decay || !aligned(a->decay, 4) || !aligned(a->beta, 4)) return fail(BIVMOE_ERR_ARGUMENT, "decay or beta: null or not aligned");
    if (!a->states || !aligned(a->states, 16) || a->stride_slot % 4 || a->stride_head % 4)
        return fail(BIVMOE_ERR_ARGUMENT, "states: null, not aligned to 16 bytes, or a stride is not a multiple of 4 values");
    if ((a->n_slots > 1 && !a->stride_slot) || (d.n_head > 1 && !a->stride_head)) return fail(BIVMOE_ERR_ARGUMENT, "states: they lie over one another");
    if (a->n_slots < 0) return fail(BIVMOE_ERR_ARGUMENT, "n_slots = %lld", (long long)a->n_slots);
    if (!a->slots || !a->first) return fail(BIVMOE_ERR_ARGUMENT, "slots or first: null pointer");
    for (const int32_t* p : {a->slots, a->first, a->past, a->keep})
        if (!aligned(p, 4)) return fail(BIVMOE_ERR_ARGUMENT, "a list of int32 is not aligned");
    const int64_t size = type_size(d.ggml_type);
    auto of = [size](const bivmoe_rows& r) { return LinearRows{(uint8_t*)r.data, r.stride_token * size, r.stride_head * size}; };
    LinearCall c{};
    c.q = of(a->q); c.k = of(a->k); c.v = of(a->v); c.out = of(a->out);
    c.decay = a->decay; c.decay_stride = a->decay_stride;
    c.beta = a->beta; c.beta_stride = a->beta_stride;
    c.states = a->states; c.slot = a->stride_slot; c.head = a->stride_head; c.n_slots = a->n_slots;
    c.slots = a->slots; c.first = a->first; c.past = a->past; c.keep = a->keep;
    c.status = l->status;
    c.n_seq = a->n_seq; c.n_tokens = a->n_tokens; c.n_head = d.n_head; c.group = d.n_head / d.n_head_qk;
    c.dim_k = d.dim_k; c.dim_v = d.dim_v; c.type = d.ggml_type;
    c.sms = l->sm_count;
    c.scale = a->scale;
    const int max_new = a->max_new && a->max_new < a->n_tokens ? a->max_new : a->n_tokens;
    DeviceScope on_device(d.device);
    cudaError_t e = cudaSuccess;
    const bool chunks = d.ggml_type == BIVMOE_BF16 && d.dim_k == 128 && d.dim_v == 128 && !c.keep && c.q.data && max_new > kSteps;
    if (!(chunks && (c.beta ? launch_linear_delta(c, (cudaStream_t)stream, &e) : launch_linear_chunks(c, max_new, (cudaStream_t)stream, &e))))
        e = launch_linear_steps(c, max_new, l->sm_count, (cudaStream_t)stream);
    return e == cudaSuccess ? BIVMOE_OK : cuda_fail(e, "bivmoe_linear_attend");
}

extern "C" int bivmoe_linear_status(bivmoe_linear* l, void* stream) {
    if (!l) return fail(BIVMOE_ERR_ARGUMENT, "null layer");
    DeviceScope on_device(l->d.device);
    cudaStream_t s = (cudaStream_t)stream;
    int32_t v = 0;
    cudaError_t e = cudaMemcpyAsync(&v, l->status, 4, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e == cudaSuccess && v) {
        e = cudaMemsetAsync(l->status, 0, 4, s);
        if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    }
    if (e != cudaSuccess) return cuda_fail(e, "bivmoe_linear_status");
    return v ? fail(BIVMOE_ERR_TIMEOUT, "a wait inside a kernel of linear attention gave up") : BIVMOE_OK;
}

// ---- the norm ----

extern "C" int bivmoe_norm(const bivmoe_norm_args* a, void* stream) {
    if (!a) return fail(BIVMOE_ERR_ARGUMENT, "null arguments");
    if (a->n_tokens < 0 || a->n_head < 1 || a->width < 1 || (int64_t)a->n_tokens * a->n_head > INT32_MAX)
        return fail(BIVMOE_ERR_ARGUMENT, "%d rows of %d heads of %d values", a->n_tokens, a->n_head, a->width);
    if (!(a->eps >= 0.0)) return fail(BIVMOE_ERR_ARGUMENT, "eps has to be zero or positive");
    const int ty = a->out.ggml_type;
    const bool q8 = ty == BIVMOE_NORM_Q8, e4m3 = ty == BIVMOE_NORM_E4M3, eight = q8 || e4m3;
    if (!is_float(ty) && !eight) return fail(BIVMOE_ERR_UNSUPPORTED, "output of type %d: F32, F16, BF16, NORM_Q8 and NORM_E4M3 have kernels", ty);
    if (q8 && a->block != 32) return fail(BIVMOE_ERR_UNSUPPORTED, "NORM_Q8 has blocks of 32, not %d", a->block);
    if (e4m3 && a->block != 0 && a->block != 128) return fail(BIVMOE_ERR_UNSUPPORTED, "NORM_E4M3 has blocks of 128 or the row (0), not %d", a->block);
    if (eight && a->block && a->width % a->block) return fail(BIVMOE_ERR_ARGUMENT, "width %d is not a multiple of the block %d", a->width, a->block);
    if (!a->n_tokens) return BIVMOE_OK;
    bool vector = a->width % 8 == 0 && aligned(a->weight, 16);
    if (!aligned(a->weight, 4)) return fail(BIVMOE_ERR_ARGUMENT, "weight: not aligned");
    NormCall c{};
    const struct { const char* name; const bivmoe_rows* r; NormRows* to; bool may_lack; } rows[] = {
        {"x", &a->x, &c.x, false}, {"add", &a->add, &c.add, true}, {"gate", &a->gate, &c.gate, true}, {"out", &a->out, &c.out, false}};
    for (const auto& x : rows) {
        if (!x.r->data && x.may_lack) continue;
        if (!x.r->data) return fail(BIVMOE_ERR_ARGUMENT, "%s: null pointer", x.name);
        const bool codes = eight && x.r == &a->out;
        if (!codes && !is_float(x.r->ggml_type)) return fail(BIVMOE_ERR_UNSUPPORTED, "%s of type %d: F32, F16 and BF16 have kernels", x.name, x.r->ggml_type);
        const int size = codes ? 1 : type_size(x.r->ggml_type);
        if (!aligned(x.r->data, size)) return fail(BIVMOE_ERR_ARGUMENT, "%s: not aligned to its type", x.name);
        *x.to = NormRows{(uint8_t*)x.r->data, x.r->stride_token * size, x.r->stride_head * size, x.r->ggml_type, size};
        const int piece = size == 1 ? 8 : 16;
        vector = vector && aligned(x.r->data, piece) && (a->n_tokens == 1 || x.to->token % piece == 0) && (a->n_head == 1 || x.to->head % piece == 0);
    }
    if (over_one_another(a->out, a->n_tokens, a->n_head) || (a->add.data && over_one_another(a->x, a->n_tokens, a->n_head)))
        return fail(BIVMOE_ERR_ARGUMENT, "out, or x with add: rows lie over one another");
    if (eight) {
        if (!a->scales || !aligned(a->scales, 4)) return fail(BIVMOE_ERR_ARGUMENT, "scales: null or not aligned");
        if (a->block && !norm_fits(a->width, vector))
            return fail(BIVMOE_ERR_UNSUPPORTED, "blocks of %d want rows of up to 16384 values, aligned to 16 bytes (codes to 8), with strides that keep it", a->block);
        if (a->out.data == a->x.data) return fail(BIVMOE_ERR_ARGUMENT, "8-bit rows cannot take the place of x");
    } else if (a->out.data == a->x.data &&
               (a->add.data || ty != a->x.ggml_type || a->out.stride_token != a->x.stride_token || a->out.stride_head != a->x.stride_head)) {
        return fail(BIVMOE_ERR_ARGUMENT, "out may be x where there is no add, with x's type and strides");
    }
    int sms = 0;
    if (int rc = device_of(a->device, "bivmoe_norm", &sms)) return rc;
    c.weight = a->weight;
    c.scales = a->scales; c.scales_stride = a->scales_stride;
    c.rows = (int64_t)a->n_tokens * a->n_head;
    c.heads = FastDiv((uint32_t)a->n_head);
    c.width = a->width; c.kind = eight ? ty : 0; c.block = a->block;
    c.eps = a->eps;
    c.per_value = 1.0 / a->width;
    DeviceScope on_device(a->device);
    const cudaError_t e = launch_norm(c, vector, sms, (cudaStream_t)stream);
    return e == cudaSuccess ? BIVMOE_OK : cuda_fail(e, "bivmoe_norm");
}

// ---- verification ----

extern "C" int bivmoe_verify(const bivmoe_verify_args* a, void* stream) {
    if (!a) return fail(BIVMOE_ERR_ARGUMENT, "null arguments");
    if (!is_float(a->ggml_type)) return fail(BIVMOE_ERR_UNSUPPORTED, "probabilities of type %d: F32, F16 and BF16 have kernels", a->ggml_type);
    if (a->vocab < 1 || a->vocab > 1 << 24) return fail(BIVMOE_ERR_ARGUMENT, "vocab %d outside 1..2^24", a->vocab);
    if (a->n_seq < 0 || a->n_seq > 65536 || a->n_tokens < 0) return fail(BIVMOE_ERR_ARGUMENT, "%d requests, %d rows", a->n_seq, a->n_tokens);
    if (!a->n_seq) return BIVMOE_OK;
    if (!a->first || !a->sample || !a->accepted || !a->token || (a->n_tokens && (!a->p || !a->tokens || !a->uniform)) || !a->length != !a->kept)
        return fail(BIVMOE_ERR_ARGUMENT, "null device pointer (length and kept go together)");
    const size_t size = type_size(a->ggml_type);
    if (!aligned(a->p, size) || !aligned(a->q, size)) return fail(BIVMOE_ERR_ARGUMENT, "p or q: not aligned to their type");
    for (const void* p : {(const void*)a->tokens, (const void*)a->first, (const void*)a->length, (const void*)a->uniform, (const void*)a->sample,
                          (const void*)a->accepted, (const void*)a->token, (const void*)a->kept})
        if (!aligned(p, 4)) return fail(BIVMOE_ERR_ARGUMENT, "a list is not aligned to 4 bytes");
    int sms = 0;
    if (int rc = device_of(a->device, "bivmoe_verify", &sms)) return rc;
    DeviceScope on_device(a->device);
    const cudaError_t e = launch_verify(*a, sms, (cudaStream_t)stream);
    return e == cudaSuccess ? BIVMOE_OK : cuda_fail(e, "bivmoe_verify");
}
