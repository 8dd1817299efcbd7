// The C ABI of the paged key/value cache: handles, checks of arguments, workspace, the choice of the
// attention kernel.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <new>
#include <vector>

#include "cache.cuh"
#include "common.cuh"

using namespace bivmoe;

struct bivmoe_cache {
    bivmoe_cache_desc d{};
    int sm_count = 0;
    RopePlan rope{};
    uint8_t* mem = nullptr;          // one allocation: parts, arrivals, the rope's tables, the status word, the count
    float* part_o = nullptr;
    float2* part_ml = nullptr;
    int32_t* arrived = nullptr;
    int32_t* status = nullptr;
    size_t arrived_bytes = 0;
    unsigned long long *unstored = nullptr, reported = 0;   // tokens without a slot so far (device); up to the last report
    // the stream of the last call that used the workspace, those of calls before it that it could not wait for
    // (they were being captured); for the end of what they did
    cudaStream_t last = nullptr;
    std::vector<cudaStream_t> behind;
    cudaEvent_t done = nullptr;
    bool used = false;
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

extern "C" void bivmoe_cache_destroy(bivmoe_cache* c) {
    if (!c) return;
    DeviceScope on_device(c->d.device);
    if (c->done) cudaEventDestroy(c->done);
    if (c->mem) cudaFree(c->mem);
    delete c;
}

extern "C" int bivmoe_cache_create(const bivmoe_cache_desc* d, bivmoe_cache** out) {
    if (out) *out = nullptr;
    if (!d || !out) return fail(BIVMOE_ERR_ARGUMENT, "null descriptor or output");
    if (d->ggml_type != BIVMOE_F16 && d->ggml_type != BIVMOE_BF16)
        return fail(BIVMOE_ERR_UNSUPPORTED, "cache type %d: F16 and BF16 have kernels", d->ggml_type);
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
        return fail(BIVMOE_ERR_UNSUPPORTED, "head_dim %d: 64, 128 and 256 have kernels", d->head_dim);
    if (d->n_head_kv < 1 || d->n_head < 1 || d->n_head > 1024 || d->n_head % d->n_head_kv)
        return fail(BIVMOE_ERR_ARGUMENT, "n_head %d (at most 1024) is not a multiple of n_head_kv %d", d->n_head, d->n_head_kv);
    if (d->page_size < 1 || d->page_size > 65536)
        return fail(BIVMOE_ERR_ARGUMENT, "page_size %d outside 1..65536", d->page_size);
    if (d->max_seqs < 1 || d->max_seqs > kCacheSeqs)
        return fail(BIVMOE_ERR_ARGUMENT, "max_seqs %d outside 1..%d", d->max_seqs, kCacheSeqs);
    if (d->max_tokens < 1 || d->max_tokens > kCacheTokens)
        return fail(BIVMOE_ERR_ARGUMENT, "max_tokens %d outside 1..%d", d->max_tokens, kCacheTokens);
    if (d->n_rot < 0 || d->n_rot > d->head_dim) return fail(BIVMOE_ERR_ARGUMENT, "n_rot %d outside 0..head_dim %d", d->n_rot, d->head_dim);
    double turns[kRopePairs];
    int32_t axis[kRopePairs];
    int pairs = 0;
    if (d->n_rot) {
        if (d->n_rot % 16) return fail(BIVMOE_ERR_UNSUPPORTED, "n_rot %d is not a multiple of 16", d->n_rot);
        if (d->rope_axes < 1 || d->rope_axes > 4) return fail(BIVMOE_ERR_ARGUMENT, "rope_axes %d outside 1..4", d->rope_axes);
        if (!(d->rope_base > 0.0) || !isfinite(d->rope_base)) return fail(BIVMOE_ERR_ARGUMENT, "rope_base has to be positive and finite");
        int sum = 0;
        for (int a = 0; a < d->rope_axes; a++) {
            if (d->rope_sections[a] < 0 || d->rope_sections[a] > d->n_rot / 2)
                return fail(BIVMOE_ERR_ARGUMENT, "rope_sections[%d] = %d outside 0..n_rot / 2", a, d->rope_sections[a]);
            sum += d->rope_sections[a];
        }
        if (sum != d->n_rot / 2) return fail(BIVMOE_ERR_ARGUMENT, "rope_sections sum to %d, not to n_rot / 2 = %d", sum, d->n_rot / 2);
        int found[4] = {};
        for (int i = 0, a = 0, end = d->rope_sections[0]; i < d->n_rot / 2; i++) {
            int of;
            if (d->rope_interleaved) {
                of = i % d->rope_axes;
                if (i >= d->rope_axes * d->rope_sections[of]) of = 0;
            } else {
                while (i >= end) end += d->rope_sections[++a];
                of = a;
            }
            found[of]++;
            axis[pairs] = of;
            turns[pairs++] = pow(d->rope_base, -2.0 * i / d->n_rot) / (2.0 * M_PI);
        }
        for (int a = 0; a < d->rope_axes; a++)
            if (found[a] != d->rope_sections[a])
                return fail(BIVMOE_ERR_ARGUMENT, "interleaved, axis %d has %d pairs and not rope_sections[%d] = %d: the sections are "
                            "too unequal", a, found[a], a, d->rope_sections[a]);
    }
    DeviceScope on_device(d->device);
    int cur = -1;
    cudaError_t e = cudaGetDevice(&cur);
    if (e == cudaSuccess && cur != d->device) e = cudaSetDevice(d->device);   // reports an invalid ordinal
    int major = 0, sms = 0;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, d->device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, d->device);
    if (e != cudaSuccess) return cuda_fail(e, "bivmoe_cache_create");
    if (major != 10)
        return fail(BIVMOE_ERR_UNSUPPORTED, "device %d is of compute capability %d.x; this library is built for sm_100a only", d->device, major);
    bivmoe_cache* c = new (std::nothrow) bivmoe_cache();
    if (!c) return fail(BIVMOE_ERR_OOM, "host allocation failed");
    c->d = *d;
    c->sm_count = sms;
    // pieces: at most two to a block (cache.cuh)
    // (none of the tcgen05 kernel's where no call has more rows than the other one's tiles)
    const size_t few = 2 * (size_t)few_blocks(d->head_dim) * c->sm_count * kFewRows,
                 tc = (int64_t)d->max_tokens * (d->n_head / d->n_head_kv) > kFewRows ? 2 * (size_t)c->sm_count * tc_rows(d->head_dim) : 0,
                 rows = few > tc ? few : tc, counts = 8 * (size_t)c->sm_count;
    size_t off = 0;
    auto take = [&off](size_t bytes) { const size_t at = off; off += (bytes + 255) & ~(size_t)255; return at; };
    const size_t o = take(rows * d->head_dim * 4), ml = take(rows * sizeof(float2)), tt = take(pairs * 8 + 8),
                 ax = take(pairs * 4 + 4), arr = take(counts * 4), st = take(16), un = take(8);
    c->arrived_bytes = counts * 4;
    e = dev_alloc((void**)&c->mem, off);
    if (e == cudaSuccess) e = cudaMemset(c->mem + arr, 0, off - arr);
    if (e == cudaSuccess && d->n_rot) e = cudaMemcpy(c->mem + tt, turns, pairs * 8, cudaMemcpyHostToDevice);
    if (e == cudaSuccess && d->n_rot) e = cudaMemcpy(c->mem + ax, axis, pairs * 4, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaEventCreateWithFlags(&c->done, cudaEventDisableTiming);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();   // the clears, before a call on any stream
    if (e != cudaSuccess) {
        const int rc = cuda_fail(e, "bivmoe_cache_create");
        bivmoe_cache_destroy(c);
        return rc;
    }
    c->part_o = (float*)(c->mem + o);
    c->part_ml = (float2*)(c->mem + ml);
    c->rope = RopePlan{d->n_rot, d->rope_adjacent, (const double*)(c->mem + tt), (const int32_t*)(c->mem + ax)};
    c->arrived = (int32_t*)(c->mem + arr);
    c->status = (int32_t*)(c->mem + st);
    c->unstored = (unsigned long long*)(c->mem + un);
    *out = c;
    return BIVMOE_OK;
}

static bool aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }

static int check_counts(const bivmoe_cache* c, int n_seq, int n_tokens) {
    if (n_seq < 0 || n_seq > c->d.max_seqs) return fail(BIVMOE_ERR_ARGUMENT, "n_seq = %d outside 0..max_seqs = %d", n_seq, c->d.max_seqs);
    if (n_tokens < 0 || n_tokens > c->d.max_tokens)
        return fail(BIVMOE_ERR_ARGUMENT, "n_tokens = %d outside 0..max_tokens = %d", n_tokens, c->d.max_tokens);
    return BIVMOE_OK;
}
static int check_pool(const char* name, const bivmoe_pool& p) {
    if (!p.data) return fail(BIVMOE_ERR_ARGUMENT, "%s: null pointer", name);
    if (p.n_pages < 0 || p.n_pages > INT32_MAX) return fail(BIVMOE_ERR_ARGUMENT, "%s: %lld pages", name, (long long)p.n_pages);
    if (!aligned(p.data, 16) || p.stride_page % 8 || p.stride_token % 8 || p.stride_head % 8)
        return fail(BIVMOE_ERR_ARGUMENT, "%s: not aligned to 16 bytes, or a stride is not a multiple of 8 values", name);
    return BIVMOE_OK;
}
static int check_table(const int32_t* table, int64_t stride, int width, int n_seq) {
    if (width < 0 || (n_seq > 1 && stride < width)) return fail(BIVMOE_ERR_ARGUMENT, "table: width %d, stride %lld", width, (long long)stride);
    if (width && !aligned(table, 4)) return fail(BIVMOE_ERR_ARGUMENT, "table: not aligned");
    if (width && n_seq && !table) return fail(BIVMOE_ERR_ARGUMENT, "table: null pointer");
    return BIVMOE_OK;
}

extern "C" int bivmoe_cache_extend(bivmoe_cache* c, const bivmoe_extend_args* a, void* stream) {
    if (!c || !a) return fail(BIVMOE_ERR_ARGUMENT, "null cache or arguments");
    if (int rc = check_counts(c, a->n_seq, a->n_tokens)) return rc;
    if (int rc = check_table(a->table, a->table_stride, a->table_width, a->n_seq)) return rc;
    if (a->n_free < 0) return fail(BIVMOE_ERR_ARGUMENT, "n_free = %d", a->n_free);
    if ((a->n_seq && (!a->past || !a->added || !a->length)) || !a->free_count || (a->n_free && !a->free_pages) || !a->first || !a->left ||
        (a->n_tokens && (!a->slots || !a->positions)))
        return fail(BIVMOE_ERR_ARGUMENT, "null device pointer");
    for (const void* p : {(const void*)a->past, (const void*)a->added, (const void*)a->held, (const void*)a->free_pages,
                          (const void*)a->free_count, (const void*)a->length, (const void*)a->first, (const void*)a->positions,
                          (const void*)a->left, (const void*)a->held_out})
        if (!aligned(p, 4)) return fail(BIVMOE_ERR_ARGUMENT, "a list of int32 is not aligned");
    if (!aligned(a->slots, 8)) return fail(BIVMOE_ERR_ARGUMENT, "slots: not aligned");
    // the blocks read the lists while the first of them writes its own
    const struct { const void* p; int64_t n; } in[] = {{a->past, a->n_seq}, {a->added, a->n_seq}, {a->held, a->n_seq}, {a->free_count, 1},
                                                       {a->free_pages, a->n_free}, {a->table, a->n_seq ? (a->n_seq - 1) * a->table_stride + a->table_width : 0}},
        out[] = {{a->length, a->n_seq}, {a->first, a->n_seq + 1}, {a->left, 2}, {a->held_out, a->n_seq}, {a->positions, a->n_tokens},
                 {a->slots, 2 * (int64_t)a->n_tokens}};
    for (const auto& i : in)
        for (const auto& o : out)
            if (i.p && o.p && (uintptr_t)i.p < (uintptr_t)o.p + 4 * o.n && (uintptr_t)o.p < (uintptr_t)i.p + 4 * i.n)
                return fail(BIVMOE_ERR_ARGUMENT, "a list that is written lies over one that is read");
    DeviceScope on_device(c->d.device);
    const cudaError_t e = launch_extend(*a, c->d.page_size, c->unstored, c->sm_count, (cudaStream_t)stream);
    return e == cudaSuccess ? BIVMOE_OK : cuda_fail(e, "bivmoe_cache_extend");
}

extern "C" int bivmoe_cache_store(bivmoe_cache* c, const bivmoe_store_args* a, void* stream) {
    if (!c || !a) return fail(BIVMOE_ERR_ARGUMENT, "null cache or arguments");
    if (int rc = check_counts(c, 0, a->n_tokens)) return rc;
    if (!a->n_tokens) return BIVMOE_OK;
    const int ty = a->q.ggml_type;
    if (ty != BIVMOE_F32 && ty != BIVMOE_F16 && ty != BIVMOE_BF16) return fail(BIVMOE_ERR_UNSUPPORTED, "rows of type %d: F32, F16 and BF16 have kernels", ty);
    if (a->k.ggml_type != ty || a->v.ggml_type != ty) return fail(BIVMOE_ERR_UNSUPPORTED, "q, k and v of different types");
    if (a->q_out.ggml_type != c->d.ggml_type) return fail(BIVMOE_ERR_ARGUMENT, "q_out is not of the cache's type");
    const size_t size = ty == BIVMOE_F32 ? 4 : 2;
    for (const bivmoe_rows* r : {&a->q, &a->k, &a->v}) {
        if (!r->data) return fail(BIVMOE_ERR_ARGUMENT, "null rows");
        if (!aligned(r->data, size)) return fail(BIVMOE_ERR_ARGUMENT, "rows are not aligned to their type");
    }
    if (!a->q_out.data || !aligned(a->q_out.data, 16) || a->q_out.stride_token % 8 || a->q_out.stride_head % 8)
        return fail(BIVMOE_ERR_ARGUMENT, "q_out: null, not aligned to 16 bytes, or a stride is not a multiple of 8 values");
    if (int rc = check_pool("k_pool", a->k_pool)) return rc;
    if (int rc = check_pool("v_pool", a->v_pool)) return rc;
    if (!a->slots || !aligned(a->slots, 8)) return fail(BIVMOE_ERR_ARGUMENT, "slots: null or not aligned");
    if (c->d.n_rot) {
        if (!a->positions || !aligned(a->positions, 4)) return fail(BIVMOE_ERR_ARGUMENT, "positions: null or not aligned");
        if (c->d.rope_axes > 1 && a->positions_stride && a->positions_stride < a->n_tokens)
            return fail(BIVMOE_ERR_ARGUMENT, "positions_stride %lld below n_tokens = %d", (long long)a->positions_stride, a->n_tokens);
    }
    DeviceScope on_device(c->d.device);
    const cudaError_t e = launch_store(*a, c->rope, c->d.ggml_type, c->d.n_head, c->d.n_head_kv, c->d.head_dim, c->d.page_size,
                                       c->sm_count, (cudaStream_t)stream);
    return e == cudaSuccess ? BIVMOE_OK : cuda_fail(e, "bivmoe_cache_store");
}

// Has s wait for what `of` has been given.  Not where `of` is captured, which cannot be waited for from outside
// the capture: `waited` is then false.
static cudaError_t wait_for(bivmoe_cache* c, cudaStream_t of, cudaStream_t s, bool& waited) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(of, &cap);
    if (e == cudaErrorStreamCaptureImplicit) {    // the legacy stream, while one that it would wait for is captured
        cudaGetLastError();
        cap = cudaStreamCaptureStatusActive;
        e = cudaSuccess;
    }
    waited = e == cudaSuccess && cap == cudaStreamCaptureStatusNone;
    if (!waited) return e;
    e = cudaEventRecord(c->done, of);
    return e == cudaSuccess ? cudaStreamWaitEvent(s, c->done, 0) : e;
}

// The workspace is one: a call on another stream than the last one's waits for what that stream had been
// given.  Not where a stream is captured: an event from outside a capture cannot be waited for in it, and one
// from inside not outside of it.  What the stream had been given before its capture is waited for by the first
// call after it.
// (An event after every call would let the last stream be destroyed in between, but it kept the next
// kernel from being scheduled early: 14.3 us a call of one token at 1000 instead of 12.)
static cudaError_t take_turn(bivmoe_cache* c, cudaStream_t s) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    const cudaError_t e = cudaStreamIsCapturing(s, &cap);
    if (e != cudaSuccess || cap != cudaStreamCaptureStatusNone) return e;
    if (c->used && c->last != s) {
        try {
            c->behind.push_back(c->last);
        } catch (const std::bad_alloc&) {
            return cudaErrorMemoryAllocation;
        }
    }
    c->last = s;
    c->used = true;
    for (size_t i = 0; i < c->behind.size();) {
        bool ordered = c->behind[i] == s;         // by the stream itself
        if (!ordered)
            if (cudaError_t f = wait_for(c, c->behind[i], s, ordered)) return f;
        if (ordered) c->behind.erase(c->behind.begin() + i);
        else i++;
    }
    return cudaSuccess;
}

static Pool pool_of(const bivmoe_pool& p) {
    return Pool{(uint8_t*)p.data, p.stride_page * 2, p.stride_token * 2, p.stride_head * 2, p.n_pages};
}

extern "C" int bivmoe_cache_attend(bivmoe_cache* c, const bivmoe_attend_args* a, void* stream) {
    if (!c || !a) return fail(BIVMOE_ERR_ARGUMENT, "null cache or arguments");
    if (int rc = check_counts(c, a->n_seq, a->n_tokens)) return rc;
    if (!a->n_tokens || !a->n_seq) return BIVMOE_OK;
    if (a->q.ggml_type != c->d.ggml_type || a->out.ggml_type != c->d.ggml_type)
        return fail(BIVMOE_ERR_ARGUMENT, "q or out is not of the cache's type");
    for (const bivmoe_rows* r : {&a->q, &a->out})
        if (!r->data || !aligned(r->data, 16) || r->stride_token % 8 || r->stride_head % 8)
            return fail(BIVMOE_ERR_ARGUMENT, "q or out: null, not aligned to 16 bytes, or a stride is not a multiple of 8 values");
    if (int rc = check_pool("k_pool", a->k_pool)) return rc;
    if (int rc = check_pool("v_pool", a->v_pool)) return rc;
    if (a->k_pool.n_pages != a->v_pool.n_pages) return fail(BIVMOE_ERR_ARGUMENT, "the pools have different numbers of pages");
    if (int rc = check_table(a->table, a->table_stride, a->table_width, a->n_seq)) return rc;
    if (!a->first || !a->length || !aligned(a->first, 4) || !aligned(a->length, 4))
        return fail(BIVMOE_ERR_ARGUMENT, "first or length: null or not aligned");
    if (a->window < 0 || a->sinks < 0) return fail(BIVMOE_ERR_ARGUMENT, "window %d or sinks %d is negative", a->window, a->sinks);
    if (!isfinite(a->scale)) return fail(BIVMOE_ERR_ARGUMENT, "scale is not finite");
    if (a->max_new < 0) return fail(BIVMOE_ERR_ARGUMENT, "max_new = %d", a->max_new);
    DeviceScope on_device(c->d.device);
    AttendCall k;
    k.q = (const uint8_t*)a->q.data;
    k.out = (uint8_t*)a->out.data;
    k.q_token = a->q.stride_token * 2; k.q_head = a->q.stride_head * 2;
    k.out_token = a->out.stride_token * 2; k.out_head = a->out.stride_head * 2;
    k.k = pool_of(a->k_pool);
    k.v = pool_of(a->v_pool);
    k.table = a->table; k.table_stride = a->table_stride; k.table_width = a->table_width;
    k.n_seq = a->n_seq; k.n_tokens = a->n_tokens;
    k.first = a->first; k.length = a->length;
    k.page = FastDiv((uint32_t)c->d.page_size);
    k.group = FastDiv((uint32_t)(c->d.n_head / c->d.n_head_kv));
    k.heads_kv = c->d.n_head_kv;
    k.window = a->window < kCachePositions ? a->window : 0;   // as wide as any length: none
    k.sinks = a->sinks < kCachePositions ? a->sinks : kCachePositions;
    k.scale_log2 = a->scale * 1.4426950408889634f;
    k.part_o = c->part_o; k.part_ml = c->part_ml; k.arrived = c->arrived; k.status = c->status;
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = take_turn(c, s);
    // Which kernel, by the most rows a request has to a kv head (max_new is the caller's word and decides the
    // speed alone: both kernels take any number).  Up to 16 rows a tile of the first reads the keys once; up to
    // 32 it reads them twice, from L2 as long as that holds them, and ends sooner with few requests or short ones.  Lengths
    // are not known here, so that two choices below are not the faster one: heads of 128, 32 rows, where many long
    // requests pass L2 by (90.2 against 82.2), and 48 rows where there are few or short ones.  Without max_new the
    // whole batch counts as one request: a decode step of 64 requests, 32 / 8 heads of 128, 249 us instead of 186.
    // us, tiles of 16 rows / tcgen05 (heads_kv 4, 4 and 2; requests x tokens):
    //   rows  heads of    1 x 300      8 x 1000     32 x 4000     4 x 20000
    //    32      64      9.9 / 13.1  13.5 / 21.1   58.4 / 67.1   41.5 / 56.8
    //    32     128     10.4 / 15.4  15.9 / 23.9   90.2 / 82.2   62.7 / 70.7
    //    32     256     11.6 / 17.8  18.3 / 27.6  100.9 / 80.5   69.7 / 113.7
    //    48     128     10.7 / 15.2  18.2 / 23.5  138.5 / 81.3   83.3 / 71.4
    const int most = a->max_new > 0 && a->max_new < a->n_tokens ? a->max_new : a->n_tokens;
    const int64_t rows = (int64_t)most * k.group.d;
    const bool few = rows <= kFewRows || (rows <= 32 && (c->d.head_dim <= 128 || (int64_t)a->n_seq * k.heads_kv <= 32));
    if (e == cudaSuccess)
        e = few ? launch_attend_few(k, c->d.head_dim, c->d.ggml_type, c->sm_count, s)
                : launch_attend_tc(k, c->d.head_dim, c->d.ggml_type, c->sm_count, s);
    return e == cudaSuccess ? BIVMOE_OK : cuda_fail(e, "bivmoe_cache_attend");
}

extern "C" int bivmoe_cache_status(bivmoe_cache* c, void* stream) {
    if (!c) return fail(BIVMOE_ERR_ARGUMENT, "null cache");
    DeviceScope on_device(c->d.device);
    int32_t word = 0;
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = cudaMemcpyAsync(&word, c->status, 4, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return cuda_fail(e, "bivmoe_cache_status");
    if (!word) return BIVMOE_OK;
    // the block that gave up did not count its part: the counts start anew
    e = cudaMemsetAsync(c->status, 0, 4, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->arrived, 0, c->arrived_bytes, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return cuda_fail(e, "bivmoe_cache_status");
    return fail(BIVMOE_ERR_TIMEOUT, "a bounded wait of the attention kernel gave up (%d)", word);
}

extern "C" int bivmoe_cache_unstored(bivmoe_cache* c, uint64_t* tokens, void* stream) {
    if (!c || !tokens) return fail(BIVMOE_ERR_ARGUMENT, "null cache or output");
    *tokens = 0;
    DeviceScope on_device(c->d.device);
    unsigned long long now = 0;           // the count is never set back: calls on other streams may be adding to it
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = cudaMemcpyAsync(&now, c->unstored, 8, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return cuda_fail(e, "bivmoe_cache_unstored");
    *tokens = now - c->reported;
    c->reported = now;
    return BIVMOE_OK;
}
